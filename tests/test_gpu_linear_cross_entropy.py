"""linear_cross_entropy and its gradients on the GPU against the formulas in 64
bits.

Tolerances. A logit is a sum of `width` products in fp32: within e = 2 width 2^-24
S of its value, S the largest sum of the products' magnitudes in its row; a loss
is within 2 e + 2^-20 (1 + the largest logit's magnitude). The gradients, element
by element: the logits' gradient dz is rounded once before both products and each
result once (u, half a step: 2^-8 bf16, 2^-11 fp16), and the probabilities inherit
the logits' errors:

  |dx| <= u (|dx| + |dz| |W|) + (4 e + 2^-16) w p |W|,  |dW| alike with |x|

with p the probabilities and w the row's weight. A probability below 2^-126 is
zero in fp32: with up to 2^12 rows and values up to 2^12 that is below 2^-100 in a
gradient."""
from __future__ import annotations

import sys

import pytest

pytestmark = pytest.mark.gpu

U = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _make(tokens, d, vocab, dtype, seed=0, ignored=0.0):
    import torch
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = getattr(torch, dtype)
    w = (torch.randn(vocab, d, generator=gen, device="cuda") * d ** -0.5).to(dt)
    targets = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    lean = torch.rand(tokens, 1, generator=gen, device="cuda") * 6
    x = (torch.randn(tokens, d, generator=gen, device="cuda") * 1.5 + lean * w[targets].float()).to(dt)
    out = torch.rand(tokens, generator=gen, device="cuda") < ignored
    return x, w, torch.where(out, -100, targets), torch.randn(tokens, generator=gen, device="cuda")


def _exact(x, w, targets, weights):
    """Losses, gradients for the rows' weights, and the bounds of all three but u."""
    import torch
    x, w, weights = x.double(), w.double(), weights.double()
    counts = targets != -100
    at = targets.clamp(min=0)[:, None]
    z = torch.where(counts[:, None], x, 0) @ w.t()
    logp = torch.log_softmax(z, 1)
    loss = torch.where(counts, -logp.gather(1, at)[:, 0], 0)
    e = 2 * x.shape[1] * 2.0 ** -24 * (torch.where(counts[:, None], x, 0).abs() @ w.abs().t()).amax(1)
    p = logp.exp()
    weights = torch.where(counts, weights, 0)[:, None]
    dz = p.scatter_add(1, at, -torch.ones_like(p[:, :1])) * weights
    loose = p * weights.abs() * (4 * e + 2.0 ** -16)[:, None]
    clean = torch.where(counts[:, None], x, 0)
    return {"loss": loss, "loss_far": 2 * e + 2.0 ** -20 * (1 + z.abs().amax(1)),
            "dx": dz @ w, "dx_mag": dz.abs() @ w.abs(), "dx_sum": loose @ w.abs(),
            "dw": dz.t() @ clean, "dw_mag": dz.abs().t() @ clean.abs(), "dw_sum": loose.t() @ clean.abs()}


def _run(x, w, targets, weights, reduction, **kw):
    import torch
    from distributedspeed_amd import linear_cross_entropy
    args = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
    loss = linear_cross_entropy(*args, targets, reduction=reduction, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, args, weights if reduction == "none" else None))


def _check(got, x, w, targets, weights, reduction, dtype):
    n = (targets != -100).sum()
    weights = weights if reduction == "none" else (weights * 0 + 1) / (n if reduction == "mean" else 1)
    e = _exact(x, w, targets, weights)
    loss, dx, dw = got
    u = U[dtype]
    if reduction == "none":
        assert ((loss.double() - e["loss"]).abs() <= e["loss_far"]).all()
    else:
        by = n if reduction == "mean" else 1
        assert abs(loss.double() - e["loss"].sum() / by) <= e["loss_far"].sum() / by + 2.0 ** -23 * loss.abs()
    for name, g in (("dx", dx), ("dw", dw)):
        bound = u * (1 + u) * (e[name].abs() + e[name + "_mag"]) + e[name + "_sum"] + 2.0 ** -100
        if dtype == "float16":
            bound = bound + 2.0 ** -25  # half of its least step
        assert g.shape == e[name].shape
        far = ((g.double() - e[name]).abs() - bound).max().item()
        assert far <= 0, (name, far)


SIZES = [(1, 64, 1000), (2, 8, 7), (3, 1, 5), (16, 63, 100), (17, 64, 129), (32, 100, 257), (33, 257, 1000), (64, 72, 5003),
         (65, 1024, 300), (100, 136, 2000), (300, 64, 70), (513, 520, 1111), (1000, 100, 3001), (3000, 256, 4000),
         (40, 64, 1), (700, 2056, 2500)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,d,vocab", SIZES)
def test_loss_and_gradients(gpu, tokens, d, vocab, dtype):
    x, w, targets, weights = _make(tokens, d, vocab, dtype, seed=tokens + d)
    _say(f"linear_cross_entropy {tokens} x {d} x {vocab} {dtype}")
    _check(_run(x, w, targets, weights, "mean"), x, w, targets, weights, "mean", dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("tokens", [5, 300])
def test_reductions_with_ignored_rows(gpu, tokens, reduction, dtype):
    """Ignored rows hold NaN and their gradients' weights too: neither is read."""
    import torch
    x, w, targets, weights = _make(tokens, 136, 900, dtype, seed=3, ignored=0.4)
    targets[0], targets[-1] = -100, 5
    skip = targets == -100
    x = torch.where(skip[:, None], float("nan"), x)
    weights = torch.where(skip, float("nan"), weights)
    got = _run(x, w, targets, weights, reduction)
    clean = [torch.where(skip, 0, weights) if t is weights else t for t in (x, w, targets, weights)]
    _check(got, *clean, reduction, dtype)
    assert not got[1][skip].any()
    if reduction == "none":
        assert not got[0][skip].any()


def test_a_vocabulary_in_pieces(gpu):
    """More bytes of logit gradients than a piece may have; the last is shorter."""
    x, w, targets, weights = _make(4096, 64, 70001, "bfloat16", seed=5, ignored=0.1)
    _say("4096 x 64 x 70001")
    _check(_run(x, w, targets, weights, "mean"), x, w, targets, weights, "mean", "bfloat16")


@pytest.mark.parametrize("d", [512, 520])
def test_the_largest_tiles(gpu, d):
    """On both sides of the width up to which the logits' gradients have smaller ones."""
    x, w, targets, weights = _make(2050, d, 20001, "float16", seed=d, ignored=0.2)
    _say(f"2050 x {d} x 20001")
    _check(_run(x, w, targets, weights, "sum"), x, w, targets, weights, "sum", "float16")


@pytest.mark.parametrize("scale", [1e-6, 1.0, 3e4])
def test_weights_of_any_scale_in_fp16(gpu, scale):
    """dz is held at a scale of its own; results below fp16's least step are zero."""
    x, w, targets, weights = _make(200, 64, 500, "float16", seed=6)
    weights = weights * scale
    loss, dx, dw = _run(x, w, targets, weights, "none")
    e = _exact(x, w, targets, weights)
    for name, g in (("dx", dx), ("dw", dw)):
        bound = U["float16"] * 1.01 * (e[name].abs() + e[name + "_mag"]) + e[name + "_sum"] + 2.0 ** -25
        fits = e[name].abs() + bound < 65504
        assert ((g.double() - e[name]).abs() <= bound)[fits].all() and fits.float().mean() > 0.5


def test_targets_of_int32_and_another_ignored_index(gpu):
    import torch
    x, w, targets, weights = _make(90, 72, 300, "bfloat16", seed=7, ignored=0.3)
    a = _run(x, w, targets, weights, "mean")
    b = _run(x, w, torch.where(targets == -100, 7_000_000, targets).int(), weights, "mean", ignore_index=7_000_000)
    c = _run(x, w, torch.where(targets == -100, 2 ** 40, targets), weights, "mean", ignore_index=2 ** 40)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and all(torch.equal(p, q) for p, q in zip(a, c))


@pytest.mark.parametrize("bad", [-1, 300, 2 ** 31, -2 ** 40])
def test_a_target_that_is_no_row(gpu, bad):
    """Its loss is NaN and so are its row's gradient and the weight's; the other
    rows' losses and gradients are theirs."""
    import torch
    x, w, targets, weights = _make(50, 72, 300, "bfloat16", seed=8)
    clean = _run(x, w, targets, weights, "none")
    targets = targets.clone()
    targets[20] = bad
    loss, dx, dw = _run(x, w, targets, weights, "none")
    keep = [i for i in range(50) if i != 20]
    assert loss[20].isnan() and torch.equal(loss[keep], clean[0][keep])
    assert dx[20].isnan().all() and torch.equal(dx[keep], clean[1][keep]) and dw.isnan().all()
    assert _run(x, w, targets, weights, "mean")[0].isnan()


def test_no_row_counts_and_no_rows(gpu):
    import torch
    from distributedspeed_amd import linear_cross_entropy
    x, w, targets, weights = _make(20, 64, 100, "bfloat16", seed=9)
    for reduction in ("mean", "sum", "none"):
        loss, dx, dw = _run(x, w, torch.full_like(targets, -100), weights, reduction)
        assert loss.isnan() if reduction == "mean" else not loss.any()
        assert not dx.any() and not dw.any()
        loss, dx, dw = _run(x[:0], w, targets[:0], weights[:0], reduction)
        assert loss.isnan() if reduction == "mean" else not loss.any()
        assert dx.shape == (0, 64) and not dw.any()
    assert linear_cross_entropy(x[:0], w, targets[:0], reduction="none").shape == (0,)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_layouts(gpu, dtype):
    """Strided and transposed x, a weight with an odd stride or address (copied),
    leading dimensions: to the bit what contiguous tensors give."""
    import torch
    from distributedspeed_amd import linear_cross_entropy
    x, w, targets, weights = _make(120, 80, 700, dtype, seed=10, ignored=0.2)
    plain = _run(x, w, targets, weights, "none")

    def padded(t, pad):
        buf = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=t.device)
        buf[:, :t.shape[1]] = t
        return buf[:, :t.shape[1]]

    odd = torch.empty(700 * 80 + 1, dtype=w.dtype, device=w.device)[1:].view(700, 80)
    odd.copy_(w)
    for a, b in ((padded(x, 3), padded(w, 8)), (x.t().contiguous().t(), padded(w, 5)), (padded(x, 16), odd),
                 (x, w.t().contiguous().t())):
        got = _run(a, b, targets, weights, "none")
        assert all(torch.equal(p, q) for p, q in zip(got, plain))
    deep = linear_cross_entropy(x.view(6, 20, 80), w, targets.view(6, 20), reduction="none")
    assert deep.shape == (6, 20) and torch.equal(deep.reshape(-1), plain[0])
    one = linear_cross_entropy(x[3], w, targets[3], reduction="none")
    assert one.shape == () and abs(one - plain[0][3]) <= 1e-5 * (1 + one)


def test_extreme_logits(gpu):
    """Logits of thousands: the loss is their difference, p is one or zero; an
    infinite or NaN logit spoils its own row's loss alone."""
    import torch
    x, w, targets, weights = _make(60, 64, 300, "bfloat16", seed=11)
    got = _run(x * 500, w, targets, weights, "none")
    _check(got, x * 500, w, targets, weights, "none", "bfloat16")
    for value in (float("nan"), float("inf")):
        bad = x.clone()
        bad[7, 5] = value
        loss, dx, _ = _run(bad, w, targets, weights, "none")
        clean = _run(x, w, targets, weights, "none")
        keep = [i for i in range(60) if i != 7]
        assert loss[7].isnan() and torch.equal(loss[keep], clean[0][keep])
        assert torch.equal(dx[keep], clean[1][keep]) and not dx[7].isfinite().all()


def test_gradients_against_differences(gpu):
    """Along a random direction, against central differences of the exact loss."""
    import torch
    x, w, targets, weights = _make(40, 72, 200, "bfloat16", seed=12, ignored=0.2)
    _, dx, dw = _run(x, w, targets, weights, "mean")
    n = (targets != -100).sum()
    e = _exact(x, w, targets, weights * 0 + 1 / n)
    gen = torch.Generator("cuda").manual_seed(1)
    h, u = 1e-4, U["bfloat16"]
    for i, (name, g) in enumerate((("dx", dx), ("dw", dw))):
        way = torch.randn(*g.shape, generator=gen, device="cuda", dtype=torch.float64)

        def loss(sign):
            moved = [x.double(), w.double()]
            moved[i] = moved[i] + sign * h * way
            return _exact(*moved, targets, weights)["loss"].sum() / n

        change = (loss(1) - loss(-1)) / (2 * h)
        slack = ((u * 1.01 * (e[name].abs() + e[name + "_mag"]) + e[name + "_sum"]) * way.abs()).sum() + 1e-5
        assert abs((g.double() * way).sum() - change) <= slack, name


def test_results_repeat_and_partial_gradients(gpu):
    import torch
    from distributedspeed_amd import linear_cross_entropy
    x, w, targets, weights = _make(500, 256, 3000, "bfloat16", seed=13, ignored=0.1)
    a, b = (_run(x, w, targets, weights, "mean") for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for i in range(2):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w))]
        g, = torch.autograd.grad(linear_cross_entropy(*args, targets), args[i])
        assert torch.equal(g, a[1 + i])
    args = [t.detach().requires_grad_(True) for t in (x, w)]
    loss = linear_cross_entropy(*args, targets)
    twice = [torch.autograd.grad(loss, args, retain_graph=True) for _ in range(2)]  # the same graph again
    assert all(torch.equal(p, q) for p, q in zip(*twice))
