"""The operators of a gated feed-forward block and of the Muon update, measured
through the public entry points. A case is a dict of plain values:

  op    "orthogonalize": a Newton-Schulz orthogonalisation of matrices
        (`shapes`: "ROWSxCOLS" or "COUNT*ROWSxCOLS", separated by spaces)
        "ffn": the gated feed-forward block over `tokens` rows of width `d`
        with `f` inner features; `train` adds its gradients
        "norm": the norms around a block with its gate and residual over
        `rows` rows of width `d`; `gate` is "none", "channel" (one value a
        channel) or "sample" (one row for `samples` equal runs of rows), `post`
        and `next` say which of the two norms are there, `train` adds gradients
  dtype the inputs' type
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS, NS_EPS, NORM_EPS = 5, 1e-7, 1e-6
BRANCH_SCALE, RESIDUAL_SCALE = 0.5, 1.0


def listed():
    ffn = {"op": "ffn", "activation": "silu"}
    norm = {"op": "norm", "post": True, "next": True}
    return [
        # The matrices of a 3-layer MLP (784-1024-1024-10), fp32 momentum.
        {"name": "muon_mlp", "op": "orthogonalize", "shapes": "1024x784 1024x1024 10x1024", "dtype": "fp32"},
        # The attention output matrices of a GPT-2-small's twelve blocks.
        {"name": "muon_gpt2_small", "op": "orthogonalize", "shapes": "12*768x768", "dtype": "bf16"},
        # A wide matrix of odd sizes in fp16.
        {"name": "muon_odd", "op": "orthogonalize", "shapes": "1001x2731", "dtype": "fp16"},
        # A Llama-3-8B up projection, taller than wide.
        {"name": "muon_llama_ffn", "op": "orthogonalize", "shapes": "14336x4096", "dtype": "bf16"},
        # One token through a Llama-3-8B block, as in serving.
        dict(ffn, name="ffn_one_token", tokens=1, d=4096, f=14336, dtype="bf16", train=False),
        # A prompt of odd length through a small block whose inner size is no multiple of eight.
        dict(ffn, name="ffn_odd_prompt", tokens=777, d=1024, f=2730, dtype="fp16", train=False, activation="gelu"),
        # A small training batch.
        dict(ffn, name="ffn_train_small", tokens=64, d=2048, f=8192, dtype="bf16", train=True),
        # A training micro-batch of a Llama-3-8B block.
        dict(ffn, name="ffn_train", tokens=4096, d=4096, f=14336, dtype="bf16", train=True),
        # One token's row, as in serving.
        dict(norm, name="norm_one_row", rows=1, d=4096, dtype="bf16", gate="channel", samples=1, train=False),
        # A training micro-batch with a per-channel gate.
        dict(norm, name="norm_train", rows=8192, d=4096, dtype="bf16", gate="channel", samples=1, train=True),
        # Odd rows and width, a gate for each of three samples, fp16.
        dict(norm, name="norm_odd", rows=3 * 1003, d=1001, dtype="fp16", gate="sample", samples=3, train=True),
        # fp32 training with no gate.
        dict(norm, name="norm_fp32", rows=2048, d=768, dtype="fp32", gate="none", samples=1, train=True),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]; a third of them are multiples of 64, a third of 8, the rest are as they fall."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    unit = rng.choice((64, 8, 1))
    return int(min(hi, max(lo, round(v / unit) * unit)))


def draw(rng):
    op = rng.choice(("orthogonalize", "ffn", "norm"))
    if op == "orthogonalize":
        n, m = _size(rng, 8, 4096), _size(rng, 8, 8192)
        if rng.random() < 0.5:
            n, m = m, n
        count = max(1, min(rng.choice((1, 2, 5, 16)), int(2 ** 25 // (n * m))))
        return {"op": op, "shapes": f"{count}*{n}x{m}", "dtype": rng.choice(("bf16", "fp16", "fp32"))}
    if op == "ffn":
        return {"op": op, "tokens": _size(rng, 1, 4096), "d": _size(rng, 64, 4096), "f": _size(rng, 64, 14336),
                "dtype": rng.choice(("bf16", "fp16")), "activation": rng.choice(("silu", "gelu")),
                "train": rng.random() < 0.5}
    samples = rng.choice((1, 2, 7))
    return {"op": op, "rows": samples * _size(rng, 1, 1024), "d": _size(rng, 64, 8192),
            "dtype": rng.choice(("bf16", "fp16", "fp32")), "gate": rng.choice(("none", "channel", "sample")),
            "samples": samples, "post": rng.random() < 0.7, "next": rng.random() < 0.7, "train": rng.random() < 0.6}


def _shapes(case):
    out = []
    for word in case["shapes"].split():
        count, _, dims = word.rpartition("*")
        n, m = dims.split("x")
        out += [(int(n), int(m))] * int(count or 1)
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * std)

    st = {"case": dict(case)}
    if case["op"] == "orthogonalize":
        # Momentum: noise with a few directions that hold about half of its norm.
        ms = []
        for n, m in _shapes(case):
            k = min(8, n, m)
            low = normal(n, k) @ normal(k, m) / math.sqrt(k)
            ms.append(((low + normal(n, m)) * 1e-3).to(dt))
        st["updates"] = ms
    elif case["op"] == "ffn":
        t, d, f = case["tokens"], case["d"], case["f"]
        st["x"] = normal(t, d).to(dt)
        st["w_gate"] = normal(f, d, std=1 / math.sqrt(d)).to(dt)
        st["w_up"] = normal(f, d, std=1 / math.sqrt(d)).to(dt)
        st["w_down"] = normal(d, f, std=1 / math.sqrt(f)).to(dt)
        if case["train"]:
            st["dy"] = normal(t, d, std=0.1).to(dt)
            for k in ("x", "w_gate", "w_up", "w_down"):
                st[k].requires_grad_(True)
    else:
        r, d = case["rows"], case["d"]
        st["residual"] = normal(r, d, std=2.0).to(dt)
        st["branch"] = normal(r, d, std=0.7).to(dt)
        st["post_weight"] = (1 + normal(d, std=0.1)).to(dt) if case["post"] else None
        st["next_weight"] = (1 + normal(d, std=0.1)).to(dt) if case["next"] else None
        gate = {"none": None, "channel": (d,), "sample": (case["samples"], d)}[case["gate"]]
        st["gate"] = None if gate is None else normal(*gate, std=0.5).to(dt)
        if case["train"]:
            st["d_hidden"] = normal(r, d, std=0.1).to(dt)
            st["d_normed"] = normal(r, d, std=0.1).to(dt) if case["next"] else None
            for k in ("residual", "branch", "post_weight", "gate", "next_weight"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
    return st


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _plain_orthogonalize(updates):
    a, b, c = COEFFICIENTS
    outs = []
    for g in updates:
        x = g.float()
        tall = x.shape[0] > x.shape[1]
        x = x.t() if tall else x
        x = x / (x.square().sum().sqrt() + NS_EPS)
        for _ in range(STEPS):
            p = x @ x.t()
            x = a * x + (b * p + c * (p @ p)) @ x
        outs.append((x.t() if tall else x).to(torch.bfloat16).contiguous())
    return outs


def _plain_act(g, name):
    """The activation and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


def _plain_ffn(st):
    case, dt = st["case"], st["x"].dtype
    x, wg, wu, wd = (st[k].detach().float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    act, slope = _plain_act(g, case["activation"])
    h = act * u
    y = (h @ wd.t()).to(dt)
    if not case["train"]:
        return {"y": y}
    dy = st["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * slope, dh * act
    return {"y": y, "dx": (dg @ wg + du @ wu).to(dt), "dw_gate": (dg.t() @ x).to(dt), "dw_up": (du.t() @ x).to(dt),
            "dw_down": (dy.t() @ h).to(dt)}


def _plain_norm(st):
    case, dt = st["case"], st["residual"].dtype
    f32 = {k: None if v is None else v.detach().float() for k, v in st.items() if k != "case"}
    r, y, w1, w2, gate = (f32[k] for k in ("residual", "branch", "post_weight", "next_weight", "gate"))
    rows, d = r.shape
    per_row = gate
    if gate is not None and gate.dim() == 2:
        per_row = gate[:, None, :].expand(-1, rows // gate.shape[0], -1).reshape(rows, d)
    rstd1 = torch.rsqrt(y.square().mean(1, keepdim=True) + NORM_EPS) if w1 is not None else None
    yhat = y * rstd1 if w1 is not None else y
    z = yhat * w1 if w1 is not None else y
    hidden = RESIDUAL_SCALE * r + BRANCH_SCALE * (z if gate is None else per_row * z)
    out = {"hidden": hidden.to(dt)}
    if w2 is not None:
        rstd2 = torch.rsqrt(hidden.square().mean(1, keepdim=True) + NORM_EPS)
        hhat = hidden * rstd2
        out["normed"] = (hhat * w2).to(dt)
    if not case["train"]:
        return out
    dh = f32["d_hidden"]
    if w2 is not None:
        dn = f32["d_normed"]
        out["d_next_weight"] = (dn * hhat).sum(0).to(dt)
        t = dn * w2
        dh = dh + rstd2 * (t - hhat * (t * hhat).mean(1, keepdim=True))
    out["d_residual"] = (RESIDUAL_SCALE * dh).to(dt)
    dz = BRANCH_SCALE * (dh if gate is None else per_row * dh)
    if gate is not None:
        dgate = BRANCH_SCALE * z * dh
        out["d_gate"] = (dgate.sum(0) if gate.dim() == 1 else dgate.view(gate.shape[0], -1, d).sum(1)).to(dt)
    if w1 is not None:
        out["d_post_weight"] = (dz * yhat).sum(0).to(dt)
        t = dz * w1
        dz = rstd1 * (t - yhat * (t * yhat).mean(1, keepdim=True))
    out["d_branch"] = dz.to(dt)
    return out


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "orthogonalize":
        if not own:
            return _plain_orthogonalize(state["updates"])
        from distributedspeed_amd.muon import orthogonalize
        return orthogonalize(state["updates"], steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    if case["op"] == "ffn":
        if not own:
            return _plain_ffn(state)
        from distributedspeed_amd.block import gated_ffn
        args = [state[k] for k in ("x", "w_gate", "w_up", "w_down")]
        y = gated_ffn(*args, activation=case["activation"])
        if not case["train"]:
            return {"y": y}
        dx, dwg, dwu, dwd = torch.autograd.grad(y, args, state["dy"])
        return {"y": y, "dx": dx, "dw_gate": dwg, "dw_up": dwu, "dw_down": dwd}
    if not own:
        return _plain_norm(state)
    from distributedspeed_amd.block import gated_residual_norm
    hidden, normed = gated_residual_norm(
        state["residual"], state["branch"], post_weight=state["post_weight"], gate=state["gate"],
        next_weight=state["next_weight"], branch_scale=BRANCH_SCALE, residual_scale=RESIDUAL_SCALE, eps=NORM_EPS)
    out = {"hidden": hidden} if normed is None else {"hidden": hidden, "normed": normed}
    if not case["train"]:
        return out
    names = [k for k in ("residual", "branch", "post_weight", "gate", "next_weight") if state[k] is not None]
    heads = [hidden] if normed is None else [hidden, normed]
    grads = [state["d_hidden"]] if normed is None else [state["d_hidden"], state["d_normed"]]
    got = torch.autograd.grad(heads, [state[k] for k in names], grads)
    out.update({"d_" + k: g for k, g in zip(names, got)})
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "orthogonalize":
        shapes = _shapes(case)
        flops = 0
        for n, m in shapes:
            s, l = min(n, m), max(n, m)
            flops += STEPS * (3 * s * s * l + s ** 3)  # the two symmetric products by halves
        return {"bytes": sum(n * m * (size + 2) for n, m in shapes), "flops": flops}
    if case["op"] == "ffn":
        t, d, f = case["tokens"], case["d"], case["f"]
        if not case["train"]:
            return {"bytes": size * (3 * d * f + 2 * t * d), "flops": 6 * t * d * f}
        return {"bytes": size * (6 * d * f + 4 * t * d), "flops": 18 * t * d * f}
    r, d = case["rows"], case["d"]
    vectors = (case["post"] + case["next"]) * d + {"none": 0, "channel": d, "sample": case["samples"] * d}[case["gate"]]
    values = (3 + case["next"]) * r * d + vectors
    if case["train"]:  # the gradients: of hidden and normed in, of residual, branch and the vectors out
        values += (3 + case["next"]) * r * d + vectors
    return {"bytes": size * values, "flops": r * d * (30 if case["train"] else 10)}


# ---- 64 bits ----------------------------------------------------------------------------------------------------------

def _exact_orthogonalize(g):
    """Every iterate is a polynomial of the first Gram matrix times the input: the polynomial is built on the short side."""
    a, b, c = COEFFICIENTS
    g = g.double()
    tall = g.shape[0] > g.shape[1]
    g = g.t().contiguous() if tall else g
    x = g / (torch.linalg.norm(g) + NS_EPS)
    gram = x.mm(x.t().contiguous())
    eye = torch.eye(gram.shape[0], dtype=torch.float64, device=g.device)
    total = eye
    for _ in range(STEPS):
        poly = a * eye + b * gram + c * gram.mm(gram)
        total = poly.mm(total)
        gram = poly.mm(gram).mm(poly)
    out = total.mm(x)
    return out.t().contiguous() if tall else out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "orthogonalize":
        return [_exact_orthogonalize(g) for g in st["updates"]]
    t = {k: v.detach().double().requires_grad_(v.requires_grad) if isinstance(v, torch.Tensor) else v
         for k, v in st.items()}
    if case["op"] == "ffn":
        act = torch.nn.functional.silu if case["activation"] == "silu" else torch.nn.functional.gelu
        args = [t[k] for k in ("x", "w_gate", "w_up", "w_down")]
        y = torch.nn.functional.linear(act(torch.nn.functional.linear(args[0], args[1]))
                                       * torch.nn.functional.linear(args[0], args[2]), args[3])
        out = {"y": y.detach()}
        if case["train"]:
            got = torch.autograd.grad(y, args, t["dy"])
            out.update(zip(("dx", "dw_gate", "dw_up", "dw_down"), got))
        return out

    def rms(v, w):
        return v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + NORM_EPS) * w

    z = t["branch"] if t["post_weight"] is None else rms(t["branch"], t["post_weight"])
    if t["gate"] is not None:
        gate = t["gate"].reshape(-1, 1, case["d"])
        z = (z.reshape(gate.shape[0], -1, case["d"]) * gate).reshape(case["rows"], case["d"])
    hidden = RESIDUAL_SCALE * t["residual"] + BRANCH_SCALE * z
    heads, grads = {"hidden": hidden}, [t.get("d_hidden")]
    if t["next_weight"] is not None:
        heads["normed"] = rms(hidden, t["next_weight"])
        grads.append(t.get("d_normed"))
    out = {k: v.detach() for k, v in heads.items()}
    if case["train"]:
        names = [k for k in ("residual", "branch", "post_weight", "gate", "next_weight") if t[k] is not None]
        got = torch.autograd.grad(list(heads.values()), [t[k] for k in names], grads)
        out.update({"d_" + k: g for k, g in zip(names, got)})
    return out
