"""gated_residual_norm and its gradients on the GPU against the formulas in 64
bits, and the block and its example as they are used together.

Tolerances, of the norm: 16-bit results are rounded once from fp32 (2^-8 for
bf16, 2^-11 for fp16, at most, an element); fp32 ones carry a dozen roundings
of 2^-24 an element and sums of up to 8192 terms or 5000 rows, added in runs
of at most a few hundred: 2^-24 * (12 + 100) = 7e-6. At a width of 1 (or 2)
the gradients through a norm are differences that cancel, which eps alone
keeps from zero: there the error is measured against their two terms."""
from __future__ import annotations

import os
import sys

import pytest

pytestmark = pytest.mark.gpu

TOL = {"bfloat16": 2.0 ** -8 + 7e-6, "float16": 2.0 ** -11 + 7e-6, "float32": 7e-6}
NAMES = ("residual", "branch", "post_weight", "gate", "next_weight")


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _make(rows, d, dtype, gate=None, post=True, nxt=True, branch=True, seed=0):
    import torch
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = getattr(torch, dtype)

    def normal(*s, std=1.0, mean=0.0):
        return (torch.randn(*s, generator=gen, device="cuda") * std + mean).to(dt)

    return {"residual": normal(rows, d, std=2.0), "branch": normal(rows, d, std=0.7) if branch else None,
            "post_weight": normal(d, std=0.1, mean=1.0) if post else None,
            "gate": None if gate is None else normal(d, std=0.5) if gate == 0 else normal(gate, d, std=0.5),
            "next_weight": normal(d, std=0.1, mean=1.0) if nxt else None,
            "d_hidden": normal(rows, d, std=0.1), "d_normed": normal(rows, d, std=0.1) if nxt else None}


def _exact(t, alpha, beta, eps, only=None):
    import torch
    x = {k: None if t[k] is None else t[k].detach().double().requires_grad_(True) for k in NAMES}

    def rms(v, w):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * w

    h = beta * x["residual"]
    if x["branch"] is not None:
        z = x["branch"] if x["post_weight"] is None else rms(x["branch"], x["post_weight"])
        if x["gate"] is not None:
            g = x["gate"].reshape(-1, 1, z.shape[1])
            z = (z.reshape(g.shape[0], -1, z.shape[1]) * g).reshape(z.shape)
        h = h + alpha * z
    heads, grads = [h], [t["d_hidden"].double()]
    if x["next_weight"] is not None:
        heads.append(rms(h, x["next_weight"]))
        grads.append(t["d_normed"].double())
    if only is not None:
        keep = [i for i in range(len(heads)) if i == only]
        pairs = [heads[i] for i in keep], [grads[i] for i in keep]
    else:
        pairs = heads, grads
    names = [k for k in NAMES if x[k] is not None]
    got = torch.autograd.grad(*pairs[:1], [x[k] for k in names], pairs[1], allow_unused=True)
    return [h.detach() for h in heads], dict(zip(names, got))


def _run(t, alpha, beta, eps):
    import torch
    from distributedspeed_amd import gated_residual_norm
    x = {k: None if t[k] is None else t[k].detach().requires_grad_(True) for k in NAMES}
    hidden, normed = gated_residual_norm(x["residual"], x["branch"], post_weight=x["post_weight"], gate=x["gate"],
                                         next_weight=x["next_weight"], branch_scale=alpha, residual_scale=beta,
                                         eps=eps)
    heads = [hidden] if normed is None else [hidden, normed]
    grads = [t["d_hidden"]] if normed is None else [t["d_hidden"], t["d_normed"]]
    names = [k for k in NAMES if x[k] is not None]
    return [h.detach() for h in heads], dict(zip(names, torch.autograd.grad(heads, [x[k] for k in names], grads)))


def _check(got, want, tol, floor=0.0):
    (gh, gg), (wh, wg) = got, want
    assert len(gh) == len(wh) and set(gg) == set(wg)
    for name, g, w in [(f"head {i}", a, b) for i, (a, b) in enumerate(zip(gh, wh))] + [(k, gg[k], wg[k]) for k in wg]:
        assert g.shape == w.shape, name
        far = (g.double() - w).norm().item()
        assert far <= tol * max(w.norm().item(), floor), (name, far, w.norm().item())


ROWS = [(1, 4096), (5, 8), (7, 9), (33, 513), (64, 1000), (130, 1001), (31, 1024), (40, 2056), (20, 4097), (12, 8192),
        (9, 8193), (6, 20001), (5000, 64)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,d", ROWS)
def test_rows_and_widths(gpu, rows, d, dtype):
    t = _make(rows, d, dtype, gate=0, seed=rows + d)
    _say(f"norm {rows}x{d} {dtype}")
    _check(_run(t, 0.5, 0.9, 1e-6), _exact(t, 0.5, 0.9, 1e-6), TOL[dtype])


@pytest.mark.parametrize("rows,d", [(6, 1), (4, 2)])
def test_widths_of_one_and_two(gpu, rows, d):
    t = _make(rows, d, "float32", gate=0, seed=3)
    # one of the two terms whose difference a gradient is: of the size of w dn / |h| and w dz / |y|
    _say(f"norm {rows}x{d}")
    _check(_run(t, 0.5, 0.9, 1e-6), _exact(t, 0.5, 0.9, 1e-6), TOL["float32"], floor=1.0)


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("nxt", [True, False])
@pytest.mark.parametrize("gate", [None, 0, 1, 3, 24])
def test_forms(gpu, post, nxt, gate):
    """With and without each norm; no gate, one of a value a channel, one row
    for all, for each of three samples, and for every row."""
    for dtype, d in (("float32", 300), ("bfloat16", 9000)):
        t = _make(24, d, dtype, gate=gate, post=post, nxt=nxt, seed=7)
        _say(f"forms {dtype} gate={gate} post={post} next={nxt}")
        _check(_run(t, -1.5, 0.25, 1e-5), _exact(t, -1.5, 0.25, 1e-5), TOL[dtype])


def test_many_samples_and_many_rows(gpu):
    """Samples of several slices each, and rows beyond one pass of the grid."""
    for rows, d, gate in ((6000, 256, 2), (9000, 64, 3000), (40000, 40, 0)):
        t = _make(rows, d, "float32", gate=gate, seed=rows)
        _say(f"{rows}x{d} gate={gate}")
        _check(_run(t, 1.0, 1.0, 1e-6), _exact(t, 1.0, 1.0, 1e-6), TOL["float32"])


def test_norm_before_a_first_block(gpu):
    t = _make(50, 600, "bfloat16", post=False, branch=False, seed=9)
    _check(_run(t, 1.0, 1.0, 1e-6), _exact(t, 1.0, 1.0, 1e-6), TOL["bfloat16"])


def test_one_output_used(gpu):
    """Only hidden, only normed, or neither carries a gradient."""
    import torch
    from distributedspeed_amd import gated_residual_norm
    t = _make(20, 333, "float32", gate=0, seed=10)
    for only in (0, 1):
        x = {k: t[k].detach().requires_grad_(True) for k in NAMES}
        heads = gated_residual_norm(x["residual"], x["branch"], post_weight=x["post_weight"], gate=x["gate"],
                                    next_weight=x["next_weight"])
        grads = torch.autograd.grad(heads[only], list(x.values()), t["d_hidden"] if only == 0 else t["d_normed"],
                                    allow_unused=True)
        want = _exact(t, 1.0, 1.0, 1e-6, only)[1]
        for k, g in zip(x, grads):
            w = want[k]
            if w is None or not bool(w.any()):
                assert g is None or not bool(g.any()), k
            else:
                assert (g.double() - w).norm().item() <= TOL["float32"] * w.norm().item(), k


def test_gradients_against_differences(gpu):
    """fp32: (L(p + e v) - L(p - e v)) / 2e against <dL/dp, v>. L's terms are
    rounded at 2^-24, so L at about 2^-24 sqrt(4000) |terms|; with e = 2^-8 the
    cubic term is of the order of e^2 = 1.5e-5. Bound: 1e-3 of the derivative,
    taken along a direction with a share of the gradient."""
    import torch
    from distributedspeed_amd import gated_residual_norm
    t = _make(12, 160, "float32", gate=3, seed=11)
    _, grads = _run(t, 0.5, 0.9, 1e-6)
    gen = torch.Generator("cuda").manual_seed(12)

    def loss(x):
        h, n = gated_residual_norm(x["residual"], x["branch"], post_weight=x["post_weight"], gate=x["gate"],
                                   next_weight=x["next_weight"], branch_scale=0.5, residual_scale=0.9)
        return (h.double() * t["d_hidden"].double()).sum() + (n.double() * t["d_normed"].double()).sum()

    for k in NAMES:
        g = grads[k].double()
        v = torch.randn(g.shape, generator=gen, device="cuda", dtype=torch.float64)
        v = v + g / g.norm() * v.norm()
        vals = []
        for e in (2.0 ** -8, -2.0 ** -8):
            p = (t[k].double() + e * v).float()
            vals += [loss({**t, k: p}).item(), (g * (p.double() - t[k].double())).sum().item()]
        diff, want = vals[0] - vals[2], vals[1] - vals[3]
        _say(f"{k}: difference {diff:.6g}, gradient {want:.6g}")
        assert abs(diff - want) <= 1e-3 * abs(want), k


def test_strides_offsets_dimensions_and_streams(gpu):
    import torch
    from distributedspeed_amd import gated_residual_norm
    t = _make(24, 200, "bfloat16", gate=2, seed=13)
    want = _exact(t, 1.0, 1.0, 1e-6)

    def padded(v, left, right):
        big = torch.full((v.shape[0], v.shape[1] + left + right), float("nan"), device="cuda", dtype=v.dtype)
        big[:, left:left + v.shape[1]] = v
        return big[:, left:left + v.shape[1]]

    rows = ("residual", "branch", "d_hidden", "d_normed")
    for left, right in ((8, 8), (1, 2), (3, 0)):
        _say(f"padding {left} {right}")
        _check(_run({**t, **{k: padded(t[k], left, right) for k in rows}}, 1.0, 1.0, 1e-6), want, TOL["bfloat16"])
    _check(_run({**t, **{k: t[k].t().contiguous().t() for k in rows}, "gate": padded(t["gate"], 1, 1)}, 1.0, 1.0, 1e-6),
           want, TOL["bfloat16"])
    first = _run(t, 1.0, 1.0, 1e-6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _run(t, 1.0, 1.0, 1e-6)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first[0], again[0]))
    assert all(torch.equal(first[1][k], again[1][k]) for k in first[1])
    h, n = gated_residual_norm(t["residual"].view(2, 12, 200), t["branch"].view(2, 12, 200), gate=t["gate"],
                               post_weight=t["post_weight"], next_weight=t["next_weight"])
    assert h.shape == n.shape == (2, 12, 200)
    assert torch.equal(h.view(24, 200), first[0][0]) and torch.equal(n.view(24, 200), first[0][1])


def test_non_finite_rows_and_zero_rows(gpu):
    """A NaN or inf stays in its row (of the row outputs); an all-zero row
    normalises to zero with finite gradients."""
    import torch
    t = _make(9, 500, "float32", gate=0, seed=14)
    clean_heads, clean = _run(t, 1.0, 1.0, 1e-6)
    bad = {**t, "branch": t["branch"].clone()}
    bad["branch"][4, 499] = float("nan")
    heads, grads = _run(bad, 1.0, 1.0, 1e-6)
    keep = [i for i in range(9) if i != 4]
    for a, b in zip(heads + [grads["residual"], grads["branch"]],
                    clean_heads + [clean["residual"], clean["branch"]]):
        assert torch.equal(a[keep], b[keep])
    assert bool(heads[0][4].isnan().all())
    zero = {**t, "branch": t["branch"].clone(), "residual": t["residual"].clone()}
    zero["branch"][2] = 0
    zero["residual"][2] = 0
    heads, grads = _run(zero, 1.0, 1.0, 1e-6)
    assert bool((heads[0][2] == 0).all()) and bool((heads[1][2] == 0).all())
    _check((heads, grads), _exact(zero, 1.0, 1.0, 1e-6), TOL["float32"])


def test_no_row_and_refusals(gpu):
    import torch
    from distributedspeed_amd import gated_residual_norm as norm
    t = _make(0, 40, "bfloat16", gate=0)
    heads, grads = _run(t, 1.0, 1.0, 1e-6)
    assert [h.shape for h in heads] == [(0, 40)] * 2
    assert all(grads[k].shape == t[k].shape and not bool(grads[k].any()) for k in grads)
    r, w = torch.ones(6, 8, device="cuda"), torch.ones(8, device="cuda")
    for args, kw, kind in (((r,), dict(gate=w), ValueError), ((r,), dict(post_weight=w), ValueError),
                           ((r, r[:3]), {}, ValueError), ((r, r), dict(post_weight=w[:4]), ValueError),
                           ((r, r), dict(next_weight=r), ValueError), ((r, r), dict(gate=torch.ones(4, 8, device="cuda")),
                                                                       ValueError),
                           ((r, r), dict(gate=torch.ones(0, 8, device="cuda")), ValueError),
                           ((r, r.half()), {}, TypeError), ((r, r), dict(gate=w.half()), TypeError),
                           ((r.cpu(), r), {}, ValueError), ((r, r.cpu()), {}, ValueError),
                           ((r.double(), r.double()), {}, TypeError), ((r, r), dict(eps=-1.0), ValueError),
                           ((r, r), dict(eps=float("nan")), ValueError), (("r",), {}, TypeError),
                           ((r[:, :0],), {}, ValueError), ((r, "y"), {}, TypeError)):
        with pytest.raises(kind):
            norm(*args, **kw)


def test_the_block_and_the_example_train(gpu):
    """GatedFFNBlock is the two operators; the example's loss falls."""
    import torch
    from distributedspeed_amd import GatedFFNBlock, gated_ffn, gated_residual_norm
    torch.manual_seed(1)
    b = GatedFFNBlock(96, 160, gate_init=0.5, branch_scale=0.7, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(33, 96, device="cuda").bfloat16()
    h, n = b(x, x)
    y = gated_ffn(x, b.w_gate, b.w_up, b.w_down)
    h2, n2 = gated_residual_norm(x, y, post_weight=b.post_weight, gate=b.gate, next_weight=b.next_weight,
                                 branch_scale=0.7)
    assert torch.equal(h, h2) and torch.equal(n, n2)
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    try:
        from train_gated_ffn import train
    finally:
        sys.path.pop(0)
    losses = train(128, 344, 3, 256, 30)
    _say(f"example: loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    assert losses[-1] < 0.8 * losses[0]
