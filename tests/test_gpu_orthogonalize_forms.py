"""orthogonalize on the GPU against the iteration in 64 bits: layouts of `out`
and of the input, step counts and coefficients, and scales. Tolerance, of the
Frobenius norm: the result's rounding to bf16 (2^-9) and three roundings of
2^-12 a step."""
from __future__ import annotations

import sys

import pytest

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _tol(steps):
    return 2.0 ** -9 + 3 * steps * 2.0 ** -12


def _exact(g, rows=(COEF,) * 5, eps=1e-7):
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / (x.norm() + eps)
    for a, b, c in rows:
        p = x.mm(x.t().contiguous())
        x = a * x + (b * p + c * p.mm(p)).mm(x)
    return x.t() if tall else x


def _far(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def _normal(shape, seed, dtype="float32", std=1.0):
    import torch
    gen = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(getattr(torch, dtype))


@pytest.mark.parametrize("n,m", [(24, 40), (90, 72)])
def test_out_with_batch_dimensions_in_any_order(gpu, n, m):
    import torch
    from distributedspeed_amd import orthogonalize
    g = _normal((2, 4, n, m), 1, "bfloat16")
    out = torch.full((4, 2, n, m), 7.0, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    _say(f"out of transposed batch dimensions, {n}x{m}")
    assert orthogonalize(g, out=out) is out
    for i in range(2):
        for j in range(4):
            assert _far(out[i, j], _exact(g[i, j])) <= _tol(5)


def test_batches_of_empty_matrices(gpu):
    import torch
    from distributedspeed_amd import orthogonalize
    for shape in ((2, 0, 4), (2, 4, 0), (2, 3, 0, 0), (0, 2, 3, 4)):
        _say(f"empty {shape}")
        assert orthogonalize(torch.ones(shape, device="cuda")).shape == shape
    good = _normal((30, 20), 2)
    got = orthogonalize([torch.ones(0, 4, device="cuda"), good, torch.ones(4, 0, device="cuda")])
    assert _far(got[1], _exact(good)) <= _tol(5)
