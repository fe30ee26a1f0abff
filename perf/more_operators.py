"""The operators of a language model's training step beside its feed-forward
blocks and optimizers, measured through the public entry points. A case is a
dict of plain values:

  op    "attention": attention over packed sequences of the given `lengths`
        ("LENGTH" or "COUNT*LENGTH", separated by spaces) with `heads` query
        heads and `kv_heads` key and value heads of `d`; `causal`; `train` adds
        the gradients. q, k and v are the parts of one projection's rows.
        "loss": the cross entropy of `tokens` rows of width `d` against a
        vocabulary of `vocab` rows, the mean over those that are not ignored
        (a share of `ignored` is) or, with a `reduction` of "none", each row's;
        `train` adds the gradients
        "rotary": the rotation of the first `dims` of `d` features of `heads`
        query and `kv_heads` key heads, in `tokens` rows at positions that
        begin at `start`; pairs lie half of `dims` apart, or side by side
        where `interleaved`; `train` adds the gradients
  dtype the inputs' type
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
IGNORE = -100
BASE = 10000.0


def listed():
    attention = {"op": "attention", "causal": True}
    loss = {"op": "loss", "ignored": 0.0, "reduction": "mean"}
    rotary = {"op": "rotary", "interleaved": False, "start": 0}
    return [
        # A short prompt through a small model's heads: latency.
        dict(attention, name="attention_short", lengths="17", heads=4, kv_heads=4, d=64, dtype="bf16", train=False),
        # One prompt through a Llama-3-8B layer's heads.
        dict(attention, name="attention_prompt", lengths="4096", heads=32, kv_heads=8, d=128, dtype="bf16", train=False),
        # A training micro-batch of that layer: documents of different lengths packed into 8192 rows.
        dict(attention, name="attention_train", lengths="2048 1777 1500 1024 777 513 300 200 53", heads=32, kv_heads=8,
             d=128, dtype="bf16", train=True),
        # Odd lengths down to one token, odd head counts, a head size between the usual ones, no causal mask.
        dict(attention, name="attention_odd", lengths="1 1003 77 2 513 5 250", heads=9, kv_heads=3, d=80, causal=False,
             dtype="fp16", train=True),
        # One long document.
        dict(attention, name="attention_long", lengths="16384", heads=16, kv_heads=2, d=64, dtype="bf16", train=True),
        # A few tokens against a small vocabulary: latency.
        dict(loss, name="loss_small", tokens=32, d=64, vocab=1000, dtype="fp16", train=True),
        # A GPT-2-small micro-batch.
        dict(loss, name="loss_gpt2_small", tokens=4096, d=768, vocab=50257, dtype="bf16", train=True),
        # An evaluation batch of odd sizes, a third of it prompt tokens that do not count: each token's loss.
        dict(loss, name="loss_odd", tokens=1777, d=1001, vocab=32003, dtype="fp16", train=False, ignored=0.33,
             reduction="none"),
        # A Llama-3-8B micro-batch, padded and prompt tokens ignored.
        dict(loss, name="loss_llama", tokens=8192, d=4096, vocab=128256, dtype="bf16", train=True, ignored=0.15),
        # One token far into a document.
        dict(rotary, name="rotary_one", tokens=1, heads=32, kv_heads=8, d=128, dims=128, dtype="bf16", train=False,
             start=131071),
        # A training micro-batch of a Llama-3-8B layer.
        dict(rotary, name="rotary_train", tokens=8192, heads=32, kv_heads=8, d=128, dims=128, dtype="bf16", train=True),
        # Odd sizes, a part of each head, pairs side by side, fp32.
        dict(rotary, name="rotary_odd", tokens=1003, heads=5, kv_heads=5, d=90, dims=34, dtype="fp32", train=True,
             interleaved=True),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]; a third of them are multiples of 64, a third of 8, the rest are as they fall."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    unit = rng.choice((64, 8, 1))
    return int(min(hi, max(lo, round(v / unit) * unit)))


def draw(rng):
    op = rng.choice(("attention", "loss", "rotary"))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4))
    if op == "attention":
        lengths = [_size(rng, 1, 4096) for _ in range(rng.choice((1, 2, 3, 5, 8)))]
        return {"op": op, "lengths": " ".join(map(str, lengths)), "heads": heads, "kv_heads": kv_heads,
                "d": rng.choice((32, 64, 72, 80, 96, 128, 128)), "causal": rng.random() < 0.8,
                "dtype": rng.choice(("bf16", "fp16")), "train": rng.random() < 0.6}
    if op == "loss":
        return {"op": op, "tokens": _size(rng, 1, 4096), "d": _size(rng, 32, 4096), "vocab": _size(rng, 100, 100000),
                "dtype": rng.choice(("bf16", "fp16")), "ignored": rng.choice((0.0, 0.0, 0.1, 0.5)),
                "reduction": rng.choice(("mean", "mean", "none")), "train": rng.random() < 0.6}
    d = rng.choice((32, 64, 80, 96, 128, 256))
    return {"op": op, "tokens": _size(rng, 1, 16384), "heads": heads, "kv_heads": kv_heads, "d": d,
            "dims": rng.choice((d, d, d // 2)), "dtype": rng.choice(("bf16", "fp16", "fp32")),
            "interleaved": rng.random() < 0.4, "start": rng.choice((0, 0, 1000, 100000)), "train": rng.random() < 0.6}


def _lengths(case):
    out = []
    for word in case["lengths"].split():
        count, _, length = word.rpartition("*")
        out += [int(length)] * int(count or 1)
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * std

    st = {"case": dict(case)}
    if case["op"] in ("attention", "rotary"):
        h, g, d = case["heads"], case["kv_heads"], case["d"]
        lengths = _lengths(case) if case["op"] == "attention" else [case["tokens"]]
        t = sum(lengths)
        rows = normal(t, h + 2 * g, d)
        rows[:, :h + g] *= 1 + normal(h + g, 1, std=0.3).abs()  # heads differ in how sharply they look
        rows = rows.to(dt)
        st["q"], st["k"], st["v"] = rows[:, :h], rows[:, h:h + g], rows[:, h + g:]
        if case["op"] == "attention":
            # What a program keeps for a batch: the plan of its lengths. The plain form's is where each row lies in a
            # batch of padded sequences.
            if own:
                from distributedspeed_amd.sequence import PackedSequences
                st["plan"] = PackedSequences(lengths, device=dev)
            else:
                n = torch.tensor(lengths, device=dev)
                at = torch.arange(int(n.max()), device=dev)
                first = n.cumsum(0) - n
                there = at[None] < n[:, None]
                st["plan"] = (torch.where(there, first[:, None] + at, 0), there)
            if case["train"]:
                st["d_out"] = normal(t, h, d, std=0.1).to(dt)
        else:
            st["positions"] = torch.arange(case["start"], case["start"] + t, device=dev)
            if case["train"]:
                st["d_q"], st["d_k"] = normal(t, h, d, std=0.1).to(dt), normal(t, g, d, std=0.1).to(dt)
        if case["train"]:
            st["q"], st["k"], st["v"] = (st[k].detach().requires_grad_(True) for k in "qkv")
        return st
    t, d, v = case["tokens"], case["d"], case["vocab"]
    st["weight"] = normal(v, d, std=1 / math.sqrt(d)).to(dt)
    targets = torch.randint(0, v, (t,), generator=gen, device=dev)
    # Hidden rows that lean towards their targets: probabilities of the target from about 1/vocab to nearly one.
    lean = 2 * math.log(v) * torch.rand(t, 1, generator=gen, device=dev)
    st["x"] = (normal(t, d, std=1.5) + lean * st["weight"][targets].float()).to(dt)
    out = torch.rand(t, generator=gen, device=dev) < case["ignored"]
    out[0] = False
    st["targets"] = torch.where(out, IGNORE, targets)
    if case["train"]:
        st["x"].requires_grad_(True)
        st["weight"].requires_grad_(True)
        if case["reduction"] == "none":
            st["d_loss"] = normal(t)
    return st


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _plain_attention(st):
    case, dt = st["case"], st["q"].dtype
    h, g, d = case["heads"], case["kv_heads"], case["d"]
    rows, there = st["plan"]
    n, s = rows.shape
    scale = 1 / math.sqrt(d)

    def padded(t):  # [tokens, heads, d] -> [sequences, kv heads, heads of a group, positions, d]
        t = t.detach().float()[rows] * there[:, :, None, None]
        return t.view(n, s, g, -1, d).permute(0, 2, 3, 1, 4).contiguous()

    def packed(t):
        return t.permute(0, 3, 1, 2, 4).reshape(n, s, -1, d)[there].to(dt)

    q, k, v = padded(st["q"]), padded(st["k"]), padded(st["v"])
    # The heads of a group side by side: one product with their key head.
    q = q.view(n, g, -1, d)
    k, v = k.view(n, g, s, d), v.view(n, g, s, d)
    scores = (q @ k.transpose(2, 3).contiguous()).view(n, g, -1, s, s) * scale
    seen = there[:, None, None, None, :]
    if case["causal"]:
        at = torch.arange(s, device=q.device)
        seen = seen & (at[:, None] >= at[None])
    scores = torch.where(seen, scores, -math.inf)
    p = torch.exp(scores - scores.amax(4, keepdim=True))
    p = p / p.sum(4, keepdim=True)
    del scores
    out = {"out": packed((p.view(n, g, -1, s) @ v).view(n, g, -1, s, d))}
    if not case["train"]:
        return out
    do = padded(st["d_out"]).view(n, g, -1, d)
    flat = p.view(n, g, -1, s)
    out["d_v"] = packed((flat.transpose(2, 3).contiguous() @ do).view(n, g, 1, s, d))
    ds = do @ v.transpose(2, 3).contiguous()
    ds = flat * (ds - (flat * ds).sum(3, keepdim=True)) * scale
    del p, flat
    out["d_q"] = packed((ds @ k).view(n, g, -1, s, d))
    out["d_k"] = packed((ds.transpose(2, 3).contiguous() @ q).view(n, g, 1, s, d))
    return out


def _plain_loss(st):
    case, dt = st["case"], st["x"].dtype
    x, w, targets = st["x"].detach().float(), st["weight"].detach().float(), st["targets"]
    counts = targets != IGNORE
    at = torch.where(counts, targets, 0)[:, None]
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    each = (torch.log(total) + top - logits.gather(1, at))[:, 0]
    n = counts.sum()
    each = torch.where(counts, each, 0)
    mean = case["reduction"] == "mean"
    out = {"loss": each.sum() / n if mean else each}
    if not case["train"]:
        return out
    dl = e / total
    dl.scatter_add_(1, at, torch.full_like(total, -1))
    dl = dl * (counts / n if mean else counts * st["d_loss"])[:, None]
    out["d_x"] = (dl @ w).to(dt)
    out["d_weight"] = (dl.t() @ x).to(dt)
    return out


def _plain_rotary(st):
    case = st["case"]
    dims = case["dims"]
    at = torch.arange(dims // 2, device=st["q"].device, dtype=torch.float64)
    angle = st["positions"].double()[:, None] * BASE ** (-2 * at / dims)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(t, sin):
        x = t.detach().float()
        a, b = (x[..., 0:dims:2], x[..., 1:dims:2]) if case["interleaved"] else (x[..., :dims // 2],
                                                                                  x[..., dims // 2:dims])
        pair = a * cos - b * sin, b * cos + a * sin
        pair = torch.stack(pair, -1).flatten(-2) if case["interleaved"] else torch.cat(pair, -1)
        return torch.cat((pair, x[..., dims:]), -1).to(t.dtype)

    out = {"q": turned(st["q"], sin), "k": turned(st["k"], sin)}
    if case["train"]:
        out.update(d_q=turned(st["d_q"], -sin), d_k=turned(st["d_k"], -sin))
    return out


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "attention":
        if not own:
            return _plain_attention(state)
        from distributedspeed_amd.sequence import packed_attention
        qkv = [state[k] for k in "qkv"]
        out = packed_attention(*qkv, state["plan"], causal=case["causal"])
        if not case["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, qkv, state["d_out"])
        return {"out": out, "d_q": dq, "d_k": dk, "d_v": dv}
    if case["op"] == "loss":
        if not own:
            return _plain_loss(state)
        from distributedspeed_amd.loss import linear_cross_entropy
        loss = linear_cross_entropy(state["x"], state["weight"], state["targets"], ignore_index=IGNORE,
                                     reduction=case["reduction"])
        if not case["train"]:
            return {"loss": loss}
        dx, dw = torch.autograd.grad(loss, [state["x"], state["weight"]], state.get("d_loss"))
        return {"loss": loss, "d_x": dx, "d_weight": dw}
    if not own:
        return _plain_rotary(state)
    from distributedspeed_amd.sequence import rotary
    q, k = rotary(state["q"], state["k"], state["positions"], base=BASE, dims=case["dims"],
                  interleaved=case["interleaved"])
    if not case["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad([q, k], [state["q"], state["k"]], [state["d_q"], state["d_k"]])
    return {"q": q, "k": k, "d_q": dq, "d_k": dk}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        h, g, d = case["heads"], case["kv_heads"], case["d"]
        lengths = _lengths(case)
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        values = 2 * (h + g) * d * sum(lengths)  # q, k, v and the output
        if case["train"]:  # the output's gradient in, q's, k's and v's out
            values *= 2
        return {"bytes": size * values, "flops": (14 if case["train"] else 4) * pairs * h * d}
    if case["op"] == "loss":
        t, d, v = case["tokens"], case["d"], case["vocab"]
        n = t - int(case["ignored"] * (t - 1))  # about how many rows count
        values = n * d + v * d
        if case["train"]:
            return {"bytes": size * (values + t * d + v * d) + 8 * t, "flops": 6 * n * d * v}
        return {"bytes": size * values + 8 * t, "flops": 2 * n * d * v}
    t, d = case["tokens"], case["d"]
    passes = 2 if case["train"] else 1
    values = 2 * (case["heads"] + case["kv_heads"]) * d * t
    return {"bytes": passes * (size * values + 8 * t), "flops": passes * 3 * values // 2 * case["dims"] // d}


# ---- 64 bits ----------------------------------------------------------------------------------------------------------

def _exact_attention(st):
    """A sequence and a head at a time, through autograd."""
    case = st["case"]
    group = case["heads"] // case["kv_heads"]
    q, k, v = (st[x].detach().double() for x in "qkv")
    out = {"out": torch.zeros_like(q)}
    if case["train"]:
        do = st["d_out"].double()
        out.update(d_q=torch.zeros_like(q), d_k=torch.zeros_like(k), d_v=torch.zeros_like(v))
    first = 0
    for n in _lengths(case):
        at = slice(first, first + n)
        first += n
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1) if case["causal"] else None
        for head in range(case["heads"]):
            args = [x[at, i].contiguous().requires_grad_(case["train"])
                    for x, i in ((q, head), (k, head // group), (v, head // group))]
            scores = args[0].mm(args[1].t()) * case["d"] ** -0.5
            if hidden is not None:
                scores = scores.masked_fill(hidden, -math.inf)
            o = torch.softmax(scores, 1).mm(args[2])
            out["out"][at, head] = o.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(o, args, do[at, head])
                out["d_q"][at, head] = dq
                out["d_k"][at, head // group] += dk
                out["d_v"][at, head // group] += dv
    return out


def _exact_loss(st):
    """Some rows at a time."""
    case, w = st["case"], st["weight"].detach().double()
    n = int((st["targets"] != IGNORE).sum())
    mean = case["reduction"] == "mean"
    weights = torch.full_like(st["targets"], 1, dtype=torch.float64) / n if mean else st.get("d_loss", st["targets"])
    each, dx, dw = [], [], torch.zeros_like(w)
    for x, targets, weight in zip(st["x"].detach().split(1024), st["targets"].split(1024), weights.split(1024)):
        x = x.double()
        logp = torch.log_softmax(x.mm(w.t()), 1)
        keep = targets.ne(IGNORE)
        hit = torch.nn.functional.one_hot(targets.clamp(min=0), w.shape[0])
        each.append(-(logp * hit).sum(1) * keep)
        if case["train"]:
            dl = (logp.exp() - hit) * (keep * weight.double())[:, None]
            dx.append(dl.mm(w))
            dw += dl.t().mm(x)
    each = torch.cat(each)
    out = {"loss": each.sum() / n if mean else each}
    if case["train"]:
        out.update(d_x=torch.cat(dx), d_weight=dw)
    return out


def _exact_rotary(st):
    """Pairs as complex numbers, turned by a unit one."""
    case = st["case"]
    dims = case["dims"]
    freq = torch.tensor([BASE ** (-2.0 * i / dims) for i in range(dims // 2)], dtype=torch.float64,
                        device=st["q"].device)
    angle = torch.outer(st["positions"].double(), freq)[:, None]
    unit = torch.polar(torch.ones_like(angle), angle)

    def turned(t, unit):
        y = t.detach().double().clone()
        pairs = y[..., :dims]
        shape = pairs.shape[:-1]
        pairs = pairs.reshape(*shape, -1, 2) if case["interleaved"] else pairs.reshape(*shape, 2, -1).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
        y[..., :dims] = (z if case["interleaved"] else z.transpose(-1, -2)).reshape(*shape, dims)
        return y

    out = {"q": turned(st["q"], unit), "k": turned(st["k"], unit)}
    if case["train"]:
        out.update(d_q=turned(st["d_q"], unit.conj()), d_k=turned(st["d_k"], unit.conj()))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "loss": _exact_loss, "rotary": _exact_rotary}[case["op"]](st)
