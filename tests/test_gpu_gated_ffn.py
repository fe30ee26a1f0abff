"""gated_ffn and its gradients on the GPU against the formulas in 64 bits.

Tolerances, of the Frobenius norm. u is half the largest relative rounding
error of the type (2^-9 for bf16, 2^-12 for fp16), which is a little above its
root mean square: the output and every gradient pass through two roundings
(h, dg or du, and the result), and a sum carries the errors of its terms at
their weight, so that 2u is what many terms that do not cancel come to. A third
u allows for short sums. Where the sums are of a handful of terms that cancel
(width 1, inner 5) the errors are measured against the sums of the terms'
magnitudes, which is what they are in proportion to. fp32 sums and the 24-bit factors are below 2^-16."""
from __future__ import annotations

import sys

import pytest

pytestmark = pytest.mark.gpu

U = {"bfloat16": 2.0 ** -9, "float16": 2.0 ** -12}


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _make(tokens, d, f, dtype, seed=0):
    import torch
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = getattr(torch, dtype)

    def normal(*s, std=1.0):
        return (torch.randn(*s, generator=gen, device="cuda") * std).to(dt)

    return (normal(tokens, d), normal(f, d, std=d ** -0.5), normal(f, d, std=d ** -0.5), normal(d, f, std=f ** -0.5),
            normal(tokens, d, std=0.1))


def _exact(x, wg, wu, wd, dy, activation):
    import torch
    F = torch.nn.functional
    act = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"), "relu": F.relu}
    args = [t.detach().double().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = F.linear(act[activation](F.linear(args[0], args[1])) * F.linear(args[0], args[2]), args[3])
    return [y.detach(), *torch.autograd.grad(y, args, dy.double())]


def _run(x, wg, wu, wd, dy, activation):
    import torch
    from distributedspeed_amd import gated_ffn
    args = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_ffn(*args, activation=activation)
    return [y.detach(), *torch.autograd.grad(y, args, dy)]


def _check(got, want, tol, scales=None):
    for name, g, w, s in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), got, want, scales or want):
        assert g.shape == w.shape, name
        far = ((g.double() - w).norm() / s.norm()).item()
        assert far <= tol, (name, far)


def _magnitudes(x, wg, wu, wd, dy):
    """The sums of the magnitudes of each result's terms (silu)."""
    import torch
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u = x @ wg.t(), x @ wu.t()
    s = torch.sigmoid(g)
    h, dh = g * s * u, dy @ wd
    dg, du = (dh * u * s * (1 + g * (1 - s))).abs(), (dh * g * s).abs()
    return [h.abs() @ wd.abs().t(), dg @ wg.abs() + du @ wu.abs(), dg.t() @ x.abs(), du.t() @ x.abs(),
            dy.abs().t() @ h.abs()]


# tokens x width x inner: one token, each small-token tile and its edges, odd
# and unaligned sizes (no multiple of 8 in one, the other, both), sums that are
# split and not, K tails inside and at a tile, several tiles each way
SIZES = [(1, 64, 64), (1, 4096, 512), (2, 8, 8), (3, 1, 5), (7, 72, 200), (16, 256, 320), (17, 65, 130), (31, 96, 1000),
         (32, 128, 127), (33, 136, 128), (64, 512, 1024), (65, 129, 64), (100, 65, 131), (128, 256, 4096),
         (129, 1024, 264), (300, 520, 1000), (513, 384, 777), (1000, 777, 384), (2048, 256, 512)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,d,f", SIZES)
def test_forward_and_gradients(gpu, tokens, d, f, dtype):
    args = _make(tokens, d, f, dtype, seed=tokens + d + f)
    _say(f"gated_ffn {tokens}x{d}x{f} {dtype}")
    _check(_run(*args, "silu"), _exact(*args, "silu"), 3 * U[dtype], _magnitudes(*args) if d * f < 8 else None)


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
def test_activations(gpu, activation):
    args = _make(96, 256, 384, "bfloat16", seed=5)
    args = (args[0] * 2, *args[1:])
    _say(activation)
    _check(_run(*args, activation), _exact(*args, activation), 3 * U["bfloat16"])


def test_large_tiles(gpu):
    """Enough tiles for the 256-tiles in every product, and sizes off them."""
    args = _make(2050, 4104, 4360, "bfloat16", seed=6)
    _say("gated_ffn 2050x4104x4360")
    _check(_run(*args, "silu"), _exact(*args, "silu"), 3 * U["bfloat16"])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,d,f", [(70, 6208, 72), (70, 72, 6216), (1100, 136, 2056), (2060, 520, 1160)])
def test_middle_tiles(gpu, tokens, d, f, dtype):
    """The 128-tiles: sums too long for the 64-tiles, which are split, along
    either size; more tiles than the 64-tiles are used for, which are not."""
    args = _make(tokens, d, f, dtype, seed=tokens + d + f)
    _say(f"gated_ffn {tokens}x{d}x{f} {dtype}")
    _check(_run(*args, "silu"), _exact(*args, "silu"), 3 * U[dtype])


@pytest.mark.parametrize("tokens,d,f,pad", [(200, 129, 260, 0), (200, 136, 261, 0), (333, 515, 1021, 3),
                                           (193, 512, 1024, 5), (260, 264, 1023, 6)])
def test_rows_off_the_chunks(gpu, tokens, d, f, pad):
    """Odd lengths and strides at enough tokens for the aligned copies, forward
    and backward, with NaN between the rows and an output gradient whose
    stride is odd too."""
    import torch
    args = _make(tokens, d, f, "bfloat16", seed=tokens + d + f + pad)
    want = _exact(*args, "silu")
    views = []
    for t in args:
        big = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), device="cuda", dtype=t.dtype)
        big[:, :t.shape[1]] = t
        views.append(big[:, :t.shape[1]])
    _say(f"gated_ffn {tokens}x{d}x{f} rows {pad} longer")
    _check(_run(*views, "silu"), want, 3 * U["bfloat16"])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,d,f", [(1, 896, 320), (2, 520, 1027), (3, 129, 2048)])
def test_few_tokens_are_rounded_once(gpu, tokens, d, f, dtype):
    """Up to three tokens' forward is as far off as the exact result rounded to
    the type: fp32 sums of a few thousand terms (relative 2^-24 each, 2^-17 at
    most) move one element in about 2^8 over a rounding boundary; bound 5%."""
    args = _make(tokens, d, f, dtype, seed=tokens + d + f)
    _say(f"gated_ffn {tokens}x{d}x{f} {dtype}")
    want = _exact(*args, "silu")[0]
    got = _run(*args, "silu")[0].double()
    once = (want.to(args[0].dtype).double() - want).norm()
    assert (got - want).norm() <= 1.05 * once


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,d,f", [(1, 896, 320), (2, 520, 1027), (3, 129, 2048), (1, 64, 8)])
def test_few_tokens_weight_gradients_are_rounded_once(gpu, tokens, d, f, dtype):
    """As above: dg, du and h enter with 16 bits (bf16) or 22, an error of 2^-8
    of the result's own rounding or less."""
    args = _make(tokens, d, f, dtype, seed=tokens + d + f)
    _say(f"gated_ffn {tokens}x{d}x{f} {dtype}")
    for name, got, want in zip(("gate", "up", "down"), _run(*args, "silu")[2:], _exact(*args, "silu")[2:]):
        once = (want.to(args[0].dtype).double() - want).norm()
        assert (got.double() - want).norm() <= 1.05 * once, name


def test_gradients_against_differences(gpu):
    """(L(p + e v) - L(p - e v)) / 2e against <dL/dp, v> for L = <y, dy>, v
    with the parameter's own scale: at e = 1/32 the cubic term is of the order
    of e^2 = 1e-3 of the derivative's size, and y's rounding (2^-12 an element,
    independent over 64 x 128 of them, over 2e) of 2^-12 * 16 / 90 = 4e-5.
    Bound: 2% of |dL/dp| |v| / sqrt(size), the derivative's standard size."""
    import torch
    from distributedspeed_amd import gated_ffn
    x, wg, wu, wd, dy = _make(64, 128, 192, "float16", seed=7)
    grads = _run(x, wg, wu, wd, dy, "silu")[1:]
    gen = torch.Generator("cuda").manual_seed(8)
    params = [x, wg, wu, wd]
    for k, name in enumerate(("x", "w_gate", "w_up", "w_down")):
        p = params[k]
        v = torch.randn(p.shape, generator=gen, device="cuda") * p.float().std()
        # a direction with a share along the gradient, so that the derivative is not a difference of noise
        g = grads[k].double()
        v = (v.double() + g / g.norm() * v.double().norm())
        vals = []
        for e in (1 / 32, -1 / 32):
            q = (p.double() + e * v).half()
            vals.append(((gated_ffn(*(q if j == k else t for j, t in enumerate(params)), activation="silu")).double()
                         * dy.double()).sum())
            step = q.double() - p.double()  # what the 16-bit parameter really moved by
            vals.append((g * step).sum())
        diff, want = (vals[0] - vals[2]).item(), (vals[1] - vals[3]).item()
        _say(f"{name}: difference {diff:.5g}, gradient {want:.5g}")
        assert abs(diff - want) <= 0.02 * abs(want), name


def test_strides_offsets_and_leading_dimensions(gpu):
    """Row-strided and offset (so 2-byte aligned) views of each operand, column
    -major weights, a 3-D input, and an output gradient that is no plain
    tensor: the same values as of contiguous copies, to the roundings' bound."""
    import torch
    from distributedspeed_amd import gated_ffn
    x, wg, wu, wd, dy = _make(90, 128, 192, "bfloat16", seed=9)
    want = _exact(x, wg, wu, wd, dy, "silu")

    def padded(t, left, right):
        big = torch.full((t.shape[0], t.shape[1] + left + right), float("nan"), device="cuda", dtype=t.dtype)
        big[:, left:left + t.shape[1]] = t
        return big[:, left:left + t.shape[1]]

    for name, views in (("row strides", [padded(t, 8, 8) for t in (x, wg, wu, wd)]),
                        ("offset by one", [padded(t, 1, 6) for t in (x, wg, wu, wd)]),
                        ("odd strides", [padded(t, 3, 2) for t in (x, wg, wu, wd)]),
                        ("column-major", [x] + [t.t().contiguous().t() for t in (wg, wu, wd)])):
        _say(name)
        _check(_run(*views, dy, "silu"), want, 3 * U["bfloat16"])
        _check(_run(*views, padded(dy, 1, 1), "silu"), want, 3 * U["bfloat16"])
    x3 = x.view(9, 10, 128).requires_grad_(True)
    y = gated_ffn(x3, wg, wu, wd)
    assert y.shape == x3.shape
    dx, = torch.autograd.grad(y, x3, dy.view(9, 10, 128).transpose(0, 1).contiguous().transpose(0, 1))
    _check([y.view(90, 128).detach(), dx.view(90, 128)], want[:2], 3 * U["bfloat16"])
    y, = (gated_ffn(x, wg, wu, wd),)
    ones = torch.autograd.grad(gated_ffn(x.requires_grad_(True), wg, wu, wd).sum(), x)[0]  # an expanded gradient
    _check([y, ones], [want[0], _exact(x, wg, wu, wd, torch.ones_like(dy), "silu")[1]], 3 * U["bfloat16"])


def test_only_the_wanted_gradients(gpu):
    import torch
    from distributedspeed_amd import gated_ffn
    x, wg, wu, wd, dy = _make(70, 64, 96, "bfloat16", seed=10)
    want = _exact(x, wg, wu, wd, dy, "silu")
    for mask in range(1, 16):
        args = [t.detach().requires_grad_(bool(mask >> k & 1)) for k, t in enumerate((x, wg, wu, wd))]
        y = gated_ffn(*args)
        y.backward(dy)
        for k, a in enumerate(args):
            if mask >> k & 1:
                assert ((a.grad.double() - want[k + 1]).norm() / want[k + 1].norm()).item() <= 3 * U["bfloat16"]
            else:
                assert a.grad is None
    y = gated_ffn(*(t.detach() for t in (x, wg, wu, wd)))
    assert not y.requires_grad
    with torch.no_grad():
        assert torch.equal(y, gated_ffn(x.requires_grad_(True), wg, wu, wd))


def test_no_token(gpu):
    import torch
    from distributedspeed_amd import gated_ffn
    args = [t.requires_grad_(True) for t in _make(0, 64, 96, "bfloat16")[:4]]
    y = gated_ffn(*args)
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y, args, torch.empty_like(y))
    assert [g.shape for g in grads] == [a.shape for a in args]
    assert all(bool((g == 0).all()) for g in grads)


def test_infinities_and_nan_stay_in_their_rows(gpu):
    """A non-finite token makes its own row of y non-finite and no other, also
    where rows share tiles and the sum over k is split or has a tail."""
    import torch
    from distributedspeed_amd import gated_ffn
    for tokens, d, f in ((3, 72, 200), (40, 520, 136), (200, 100, 300)):
        x, wg, wu, wd, dy = _make(tokens, d, f, "bfloat16", seed=tokens)
        clean = gated_ffn(x, wg, wu, wd)
        bad = x.clone()
        bad[1, d - 1] = float("nan")
        _say(f"NaN in one of {tokens} tokens")
        y = gated_ffn(bad, wg, wu, wd)
        assert bool(y[1].isnan().all())
        keep = [i for i in range(tokens) if i != 1]
        assert torch.equal(y[keep], clean[keep])
        bad[1, d - 1] = float("inf")
        y = gated_ffn(bad, wg, wu, wd)
        assert not bool(y[1].isfinite().all()) and torch.equal(y[keep], clean[keep])
        args = [bad.detach().requires_grad_(True), wg, wu, wd]
        dx, = torch.autograd.grad(gated_ffn(*args), args[0], dy)
        ref, = torch.autograd.grad(gated_ffn(x.detach().requires_grad_(True), wg, wu, wd), x, dy, allow_unused=True) \
            if x.requires_grad else (None,)
        assert bool(dx[keep].isfinite().all()) and ref is None


def test_repeats_bit_for_bit_other_stream_and_graph(gpu):
    import torch
    from distributedspeed_amd import gated_ffn
    x, wg, wu, wd, dy = _make(48, 256, 1024, "bfloat16", seed=12)
    first, again = _run(x, wg, wu, wd, dy, "silu"), _run(x, wg, wu, wd, dy, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = _run(x, wg, wu, wd, dy, "silu")
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, again, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gated_ffn(x, wg, wu, wd)
    for k in range(3):
        _say(f"replay {k}")
        fresh = _make(48, 256, 1024, "bfloat16", seed=30 + k)[0]
        want = gated_ffn(fresh, wg, wu, wd)
        x.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(gpu):
    import torch
    from distributedspeed_amd import GatedFFNBlock, gated_ffn
    x, wg, wu, wd, _ = _make(4, 16, 24, "bfloat16")
    for args, kind in (((x, wg, wu[:-1], wd), ValueError), ((x, wg, wu, wd.t()), ValueError),
                       ((x[:, :8], wg, wu, wd), ValueError), ((x, wg[0], wu, wd), ValueError),
                       ((x, wg.half(), wu, wd), TypeError), ((x.float(), wg, wu, wd), TypeError),
                       ((x, wg.cpu(), wu, wd), ValueError), ((x.cpu(), wg, wu, wd), ValueError),
                       (("x", wg, wu, wd), TypeError), ((x, None, wu, wd), TypeError),
                       ((x, wg[:0], wu[:0], wd[:, :0]), ValueError)):
        with pytest.raises(kind):
            gated_ffn(*args)
    with pytest.raises(ValueError):
        gated_ffn(x, wg, wu, wd, activation="tanh")
    with pytest.raises(ValueError):
        GatedFFNBlock(8, 8, activation="tanh")
    y = gated_ffn(x.requires_grad_(True), wg, wu, wd)
    g, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
