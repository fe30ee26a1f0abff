"""rotary and its gradient on the GPU against the formula in 64 bits.

Tolerance, element by element: the result is rounded once (u, half a step of the
type: 2^-8, 2^-11, 2^-24); the cosine and sine are fp32 values of angles that are
within 2^-22 of a turn, the products and their sum fp32: 2^-19 (|a| + |b|). Below
2^-14 fp16's step is 2^-24 whatever the value: half of it there."""
from __future__ import annotations

import math
import sys

import pytest

pytestmark = pytest.mark.gpu

U = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _exact(x, positions, base, dims, interleaved, sign=1):
    """(the result, |a| + |b| of each element's pair)"""
    import torch
    y = x.double().clone()
    mag = y.abs()
    half = dims // 2
    if half:
        i = torch.arange(half, device=x.device, dtype=torch.float64)
        angle = sign * positions.double()[..., None, None] * torch.exp(i * (-2 * math.log(base) / dims))
        at = [slice(0, dims, 2), slice(1, dims, 2)] if interleaved else [slice(0, half), slice(half, dims)]
        a, b = (x.double()[..., s] for s in at)
        y[..., at[0]] = a * angle.cos() - b * angle.sin()
        y[..., at[1]] = b * angle.cos() + a * angle.sin()
        for s in at:
            mag[..., s] = a.abs() + b.abs()
    return y, mag


def _check(got, x, positions, base, dims, interleaved, sign=1):
    want, mag = _exact(x, positions, base, dims, interleaved, sign)
    u = U[str(got.dtype).split(".")[1]]
    assert got.shape == x.shape and got.dtype == x.dtype
    least = 2.0 ** -25 if got.dtype.itemsize == 2 and u == U["float16"] else 0.0
    assert ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -19 * mag + least).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,dims", [(1, 4, 1, 64, 64), (3, 1, 1, 2, 2), (7, 5, 3, 80, 34),
                                                         (65, 2, 2, 128, 128), (130, 3, 1, 33, 14), (40, 2, 1, 256, 0),
                                                         (9, 1, 2, 1024, 1024), (1000, 8, 2, 96, 48), (5, 2, 2, 7, 6)])
def test_forward_and_gradient(gpu, tokens, heads, kv_heads, d, dims, interleaved, dtype):
    import torch
    from distributedspeed_amd import rotary
    gen = torch.Generator("cuda").manual_seed(tokens + d)
    dt = getattr(torch, dtype)

    def normal(h):
        return torch.randn(tokens, h, d, generator=gen, device="cuda").to(dt)

    q, k, gq, gk = normal(heads).requires_grad_(True), normal(kv_heads).requires_grad_(True), normal(heads), normal(kv_heads)
    positions = torch.randint(-5000, 200000, (tokens,), generator=gen, device="cuda")
    _say(f"rotary {tokens} x {heads}/{kv_heads} x {d}, {dims} turned, {dtype}")
    y, z = rotary(q, k, positions, dims=dims, interleaved=interleaved)
    _check(y.detach(), q.detach(), positions, 10000.0, dims, interleaved)
    _check(z.detach(), k.detach(), positions, 10000.0, dims, interleaved)
    dq, dk = torch.autograd.grad([y, z], [q, k], [gq, gk])
    _check(dq, gq, positions, 10000.0, dims, interleaved, -1)
    _check(dk, gk, positions, 10000.0, dims, interleaved, -1)


@pytest.mark.parametrize("base", [10000.0, 500000.0, 1.0, 0.5])
def test_far_positions_and_bases(gpu, base):
    """Up to 2^31 - 1 and down to -2^31, as int32 and int64: fp32 angles would be
    off by whole turns. With 53 bits, 2^31 radians are within 2^-22."""
    import torch
    from distributedspeed_amd import rotary
    positions = torch.tensor([0, 1, -1, 131071, 2 ** 24 + 1, 2 ** 30, 2 ** 31 - 1, -2 ** 31], device="cuda")
    q = torch.randn(8, 2, 64, device="cuda")
    a, b = rotary(q, q[:, :1], positions, base=base)
    c, _ = rotary(q, q[:, :1], positions.int(), base=base)
    assert torch.equal(a, c)
    if base >= 1:
        _check(a, q, positions, base, 64, False)
        _check(b, q[:, :1], positions, base, 64, False)


def test_the_gradient_against_differences(gpu):
    """The map is linear: its value at a difference is the difference of its
    values, and the gradient's product with a direction is that of the output's
    gradient with the map of it (fp32: 4096 terms of 2^-20)."""
    import torch
    from distributedspeed_amd import rotary
    q, k, way, g = (torch.randn(32, 2, 64, device="cuda") for _ in range(4))
    positions = torch.arange(32, device="cuda")
    x = q.clone().requires_grad_(True)
    y, _ = rotary(x, k, positions)
    dx, = torch.autograd.grad(y, x, g)
    moved = rotary(q + way, k, positions)[0].double() - rotary(q - way, k, positions)[0].double()
    scale = (dx.abs() * way.abs()).sum().double() + (g.abs() * way.abs()).sum().double()
    assert abs((dx.double() * way.double()).sum() - (g.double() * moved).sum() / 2) <= 2.0 ** -18 * scale


def test_layouts_leading_dimensions_and_partial_gradients(gpu):
    import torch
    from distributedspeed_amd import rotary
    rows = torch.randn(6, 50, 4 + 2, 40, device="cuda").bfloat16()
    positions = torch.arange(50, device="cuda").expand(6, 50)
    q, k = rows[:, :, :4], rows[:, :, 4:]
    y, z = rotary(q, k, positions, dims=30)
    assert y.shape == q.shape and y.is_contiguous()
    _check(y, q, positions, 10000.0, 30, False)
    _check(z, k, positions, 10000.0, 30, False)
    turned = torch.empty(4, 40, 300, device="cuda", dtype=torch.bfloat16)  # features outermost
    turned.copy_(q.reshape(300, 4, 40).permute(1, 2, 0))
    odd = torch.empty(300 * 80 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(300, 2, 40)
    odd.copy_(k.reshape(300, 2, 40))
    a, b = rotary(turned.permute(2, 0, 1), odd, positions.reshape(-1), dims=30)
    assert torch.equal(a, y.view(300, 4, 40)) and torch.equal(b, z.view(300, 2, 40))
    for i in range(2):  # one of the two alone
        args = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate((q, k))]
        out = rotary(*args, positions, dims=30)
        g = torch.randn_like(out[i])
        d, = torch.autograd.grad(out[i], args[i], g)
        _check(d, g, positions, 10000.0, 30, False, -1)
    both = [t.detach().clone().requires_grad_(True) for t in (q, k)]
    out = rotary(*both, positions)
    d, = torch.autograd.grad(out[1].float().sum(), both[1], retain_graph=True)
    _check(d, torch.ones_like(d), positions, 10000.0, 40, False, -1)
    none, = torch.autograd.grad(out[1].float().sum(), both[0], allow_unused=True)
    assert none is None or not none.any()


def test_values_that_are_not_finite_and_no_rows(gpu):
    import torch
    from distributedspeed_amd import rotary
    q = torch.randn(4, 2, 32, device="cuda").half()
    positions = torch.arange(4, device="cuda")
    clean, _ = rotary(q, q, positions)
    bad = q.clone()
    bad[1, 0, 3] = float("nan")
    got, _ = rotary(bad, q, positions)
    assert got[1, 0, 3].isnan() and got[1, 0, 19].isnan()
    got[1, 0, 3], got[1, 0, 19] = clean[1, 0, 3], clean[1, 0, 19]
    assert torch.equal(got, clean)
    x = torch.empty(0, 2, 32, device="cuda").requires_grad_(True)
    y, z = rotary(x, x, positions[:0])
    (y.sum() + z.sum()).backward()
    assert y.shape == (0, 2, 32) and x.grad.shape == (0, 2, 32)


def test_as_many_rows_as_there_may_be(gpu):
    """2^27: a block then takes several runs of rows."""
    import torch
    from distributedspeed_amd import rotary
    n = 2 ** 27
    gen = torch.Generator("cuda").manual_seed(0)
    q = torch.randn(n, 1, 2, generator=gen, device="cuda", dtype=torch.float16)
    k = q.view(n, 2, 1)[:, :1].expand(-1, 1, 2)
    positions = torch.arange(n, dtype=torch.int32, device="cuda") % 1000
    got = rotary(q, k, positions)
    for first in (0, 2 ** 25 - 500, 2 ** 26 - 500, n - 1000):
        at = slice(first, first + 1000)
        for x, y in zip(got, (q, k)):
            _check(x[at], y[at], positions[at], 10000.0, 2, False)
