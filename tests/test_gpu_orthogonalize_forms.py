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


def _spectrum(n, m, values, seed, dtype="float32"):
    """An n x m matrix with these singular values."""
    import torch
    u = torch.linalg.qr(_normal((n, n), seed, "float64"))[0][:, :len(values)]
    v = torch.linalg.qr(_normal((m, len(values)), seed + 1, "float64"))[0]
    return (u * torch.as_tensor(values, device="cuda", dtype=torch.float64)).mm(v.t().contiguous()).to(getattr(torch, dtype))


POLAR = (2.0, -1.5, 0.5)  # converges to the polar factor


@pytest.mark.parametrize("steps,coef", [(5, COEF), (6, COEF), (8, COEF), (10, COEF), (12, COEF), (20, COEF),
                                        (12, POLAR), (20, POLAR), (40, POLAR), (24, (1.5, -0.5, 0.0))])
@pytest.mark.parametrize("n,m,spread", [(64, 64, 3), (48, 200, 4), (200, 48, 4), (13, 40, 3), (64, 1000, 0), (7, 1, 0)])
def test_any_number_of_steps_of_a_short_side(gpu, n, m, spread, steps, coef):
    """Sides of at most 64, singular values spread over 10^0 to 10^4. A numpy
    model of the runs of steps in fp32 is at most 1.3e-3 off (twenty steps of
    Muon's coefficients, 10^3) and 4e-4 to twelve: bound 2^-9 for the result's
    bf16 and twice that."""
    import torch
    from distributedspeed_amd import orthogonalize
    k = min(n, m)
    values = [10.0 ** (-spread * i / max(1, k - 1)) for i in range(k)] if spread else None
    g = _normal((n, m), n + m) if values is None else (_spectrum(n, m, values, n + m) if n <= m else
                                                       _spectrum(m, n, values, n + m).t().contiguous())
    _say(f"{n}x{m} over 10^{spread}, {steps} steps of {coef}")
    got = orthogonalize(g, steps=steps, coefficients=coef)
    assert bool(got.isfinite().all())
    assert _far(got, _exact(g, (coef,) * steps)) <= 2.0 ** -9 + (2.6e-3 if steps > 12 else 2.0 ** -10)


@pytest.mark.parametrize("steps", [5, 8, 12, 20, 64])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,m", [(64, 64), (40, 300), (300, 40), (33, 64)])
def test_a_rank_of_four_at_any_number_of_steps(gpu, n, m, dtype, steps):
    """Rows of zeros stay zeros and the rest is as exact as ever. Of random
    factors the null space holds the input's rounding (2^-24 of its norm),
    which 3.44^steps multiplies: at 8 steps 7e-4 of the result (modelled), at
    12 a tenth, then as large as the rest, but bounded by the iteration, whose
    singular values stay below 1.21; what lies in the matrix's own space is
    exact to the result's rounding at any count."""
    import torch
    from distributedspeed_amd import orthogonalize
    g = torch.zeros(n, m, device="cuda", dtype=getattr(torch, dtype))
    g[5:9] = _normal((4, m), 11, dtype)
    _say(f"four rows of {n}x{m} {dtype}, {steps} steps")
    want = _exact(g, (COEF,) * steps)
    got = orthogonalize(g, steps=steps)
    assert _far(got, want) <= 2.0 ** -9 + (2.0 ** -10 if steps <= 20 else 2.0 ** -8)
    assert bool((got[:5] == 0).all()) and bool((got[9:] == 0).all())
    a, b = _normal((n, 4), 12), _normal((4, m), 13)
    g = a.mm(b)
    want, got = _exact(g, (COEF,) * steps), orthogonalize(g, steps=steps)
    _say("random factors")
    assert bool(got.isfinite().all()) and torch.linalg.matrix_norm(got.float(), 2).item() <= 1.25
    if steps <= 8:
        assert _far(got, want) <= 2.0 ** -9 + 2.0 ** -9
    u, v = torch.linalg.qr(a.double())[0], torch.linalg.qr(b.t().double().contiguous())[0]
    if steps <= 20:
        inside = [u.t().contiguous().mm(t.double()).mm(v) for t in (got, want)]
        assert _far(*inside) <= 2.0 ** -8


def test_muon_steps_of_many_iterations(gpu):
    """A rank-four grad for matrices with a short side, 12 iterations a step:
    the update is bounded as the iteration is."""
    import torch
    from distributedspeed_amd import MuonOptimizer
    ps = [torch.nn.Parameter(_normal(s, 20, std=0.05)) for s in ((64, 64), (30, 100), (100, 30))]
    before = [p.detach().clone() for p in ps]
    opt = MuonOptimizer(ps, lr=0.01, weight_decay=0.0, ns_steps=12, adjust_lr="original")
    for p in ps:
        p.grad = _normal((p.shape[0], 4), 21).mm(_normal((4, p.shape[1]), 22))
    _say("muon, 12 iterations")
    opt.step()
    for p, w in zip(ps, before):
        factor = 0.01 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        o = (w - p.detach()).double() / factor
        assert bool(p.isfinite().all()) and torch.linalg.matrix_norm(o, 2).item() <= 1.25
        g = p.grad.double()
        u, _, v = torch.linalg.svd(g, full_matrices=False)
        u, v = u[:, :4].contiguous(), v[:4].contiguous()
        want = _exact(p.grad * 0.0975, (COEF,) * 12)  # (1 - mu^2) g of a first Nesterov step
        inside = [u.t().contiguous().mm(t).mm(v.t().contiguous()) for t in (o, want)]
        assert _far(*inside) <= 2.0 ** -8


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,m", [(64, 1024), (1024, 40), (16, 16), (5, 3000), (96, 200), (300, 130)])
def test_scale_does_not_matter_at_either_end(gpu, n, m, dtype):
    """Entries from 1e-30 to 1e37 (their squares leave fp32's range from 1e-19
    down and 1e19 up), in a list and alone, eps far below or, at 1e-19 and
    below, beside and above the norm. A short side takes a power of two out, so
    that its bits are the scaled matrix's own. With a longer one the iterates
    are fp16 times 4096: where the norm is far below eps, they lose bits to
    their range, so that those scales are left to the short sides."""
    import torch
    from distributedspeed_amd import orthogonalize
    base = _normal((n, m), 31, dtype).clamp_(-8, 8)
    small = min(n, m) <= 64
    for power in (-100, -80, -67, -63, -40, 40, 63, 80, 120):
        if not small and power < -50:
            continue
        g = (base.double() * 2.0 ** power).to(base.dtype)
        _say(f"{n}x{m} {dtype} times 2^{power}")
        got = orthogonalize(g, eps=1e-20)
        assert bool(got.isfinite().all())
        want = _exact(g, eps=1e-20)
        if want.norm() > 1e-30:  # of bf16's range
            assert _far(got, want) <= _tol(5)
    if small:
        a, b = orthogonalize(base, eps=2.0 ** -60), orthogonalize((base.double() * 2.0 ** 30).to(base.dtype), eps=2.0 ** -30)
        assert torch.equal(a, b)
    both = orthogonalize([base, (base.double() * 2.0 ** 110).to(base.dtype), torch.zeros_like(base)])
    assert _far(both[0], _exact(base)) <= _tol(5) and _far(both[1], _exact(base)) <= _tol(5) and not bool(both[2].any())


def test_one_large_value_among_small_ones(gpu):
    """The parts of a long side at scales of their own: a column of 1e30 and
    one of 1e-30 in different ones, and an infinity or a NaN at any place."""
    import torch
    from distributedspeed_amd import orthogonalize
    for n, m in ((20, 5000), (5000, 20)):
        for at in (0, 2500, 4999):
            g = _normal((n, m), 41, std=1e-30)
            (g if n < m else g.t())[:, at] *= 1e30
            _say(f"{n}x{m}, 1e30 times at {at}")
            # rank one but for 1e-30: the rest is below the result's last bit
            assert _far(orthogonalize(g), _exact(g)) <= _tol(5)
            for bad in (float("inf"), float("nan"), -float("inf")):
                h = g.clone()
                (h if n < m else h.t())[7, at] = bad
                assert bool(orthogonalize(h).isnan().all())


def test_muon_steps_with_grads_at_the_ends_of_fp32(gpu):
    """A finite grad is no overflow, whatever the shorter side."""
    import torch
    from distributedspeed_amd import MuonOptimizer
    for power, skipped in ((100, False), (-60, False)):
        ps = [torch.nn.Parameter(_normal(s, 50, std=0.05)) for s in ((64, 256), (130, 100))]
        before = [p.detach().double() for p in ps]
        opt = MuonOptimizer(ps, lr=0.01, weight_decay=0.0, eps=1e-20)
        for p in ps:
            p.grad = _normal(p.shape, 51) * 2.0 ** power
        _say(f"grads times 2^{power}")
        opt.step()
        assert opt.last_step_skipped() == skipped
        for p, w in zip(ps, before):
            factor = 0.01 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            o = (w - p.detach().double()) / factor
            want = _exact(p.grad * 0.0975, eps=1e-20)
            # fp32's rounding of weights of 0.05 in units of the update
            assert (o - want).norm() <= 15 * 2.0 ** -12 * want.norm() + 1e-6 * w.norm() / factor


def test_a_list_in_several_runs_of_scratch(gpu):
    """Five matrices whose scratch is more than a run's, small ones among them."""
    import torch
    from distributedspeed_amd import orthogonalize
    big = [_normal(s, 60 + k, "bfloat16") for k, s in enumerate(((4096, 6000), (6000, 4096)) * 2 + ((4096, 6000),))]
    small = [_normal((30, 50), 70 + k, "bfloat16") for k in range(3)] + [_normal((90, 70), 80, "bfloat16")]
    ms = [big[0], small[0], big[1], small[3], big[2], small[1], big[3], small[2], big[4]]
    _say("five of 4096 x 6000")
    for g, o in zip(ms, orthogonalize(ms)):
        assert o.shape == g.shape and _far(o, _exact(g)) <= _tol(5)
