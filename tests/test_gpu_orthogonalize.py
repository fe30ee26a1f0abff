"""orthogonalize and MuonOptimizer on the GPU against the iteration in 64 bits.

Tolerances. The result is bf16: rounding an element moves it by at most 2^-9
of itself, so at most 2^-9 of the result's Frobenius norm in all. Before it, a
step rounds A, B and X to fp16 once each (2^-12 of an element at most): 15
roundings in five steps, none of which the later steps expand more than the
result itself. Bound: 2^-9 + 15 * 2^-12 = 5.6e-3 of the norm. The momentum is
fp32: three operations of 2^-24 each a step, on terms of either sign."""
from __future__ import annotations

import math
import sys

import pytest

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
TOL = 2.0 ** -9 + 15 * 2.0 ** -12


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _exact(g, rows=(COEF,) * 5, eps=1e-7):
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.square().sum().sqrt() + eps)
    for a, b, c in rows:
        p = x.mm(x.t().contiguous())
        x = a * x + (b * p + c * p.mm(p)).mm(x.contiguous())
    return x.t() if tall else x


def _far(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def _matrix(gen, n, m, dtype, std=1e-3, device="cuda"):
    import torch
    return (torch.randn(n, m, generator=gen, device=device) * std).to(dtype)


def _gen(seed=0):
    import torch
    return torch.Generator("cuda").manual_seed(seed)


SHAPES = [(1, 1), (1, 7), (9, 1), (8, 8), (13, 40), (63, 65), (64, 64), (65, 200), (200, 65), (127, 129), (128, 512),
          (257, 255), (300, 1001), (1001, 300), (777, 2050), (1536, 1536)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,m", SHAPES)
def test_one_matrix(gpu, n, m, dtype):
    import torch
    from distributedspeed_amd import orthogonalize
    g = _matrix(_gen(n * 10007 + m), n, m, getattr(torch, dtype))
    _say(f"orthogonalize {n}x{m} {dtype}")
    got = orthogonalize(g)
    assert got.shape == g.shape and got.dtype == torch.bfloat16 and got.is_contiguous()
    assert _far(got, _exact(g)) <= TOL


def test_large_tiles_and_a_long_side(gpu):
    """Sizes that take the 128-, 192- and 256-tiles, and a side of 20000."""
    import torch
    from distributedspeed_amd import orthogonalize
    for n, m in ((2304, 5000), (2100, 6016), (6016, 2100), (4100, 4104), (24, 20000)):
        g = _matrix(_gen(n), n, m, torch.bfloat16)
        _say(f"orthogonalize {n}x{m}")
        assert _far(orthogonalize(g), _exact(g)) <= TOL


def test_a_list_of_any_shapes_is_each_matrix_alone(gpu):
    """More matrices than one launch's table holds, both orientations, empty
    ones among them: the same bits as one call each where the tiles agree, and
    within the bound of the exact result in any case."""
    import torch
    from distributedspeed_amd import orthogonalize
    gen = _gen(3)
    sizes = [(5 + 7 * k % 90, 3 + 11 * k % 130) for k in range(61)] + [(0, 5), (4, 0), (700, 300), (300, 700)]
    ms = [_matrix(gen, n, m, torch.float32, std=10.0 ** (k % 7 - 3)) for k, (n, m) in enumerate(sizes)]
    _say(f"list of {len(ms)}")
    for g, o in zip(ms, orthogonalize(ms)):
        assert o.shape == g.shape
        if g.numel():
            assert _far(o, _exact(g)) <= TOL


def test_stacked_strided_and_transposed_inputs(gpu):
    import torch
    from distributedspeed_amd import orthogonalize
    gen = _gen(4)
    stack = torch.randn(2, 3, 40, 56, generator=gen, device="cuda").bfloat16()
    _say("stack")
    got = orthogonalize(stack)
    assert got.shape == stack.shape
    for i in range(2):
        for j in range(3):
            assert _far(got[i, j], _exact(stack[i, j])) <= TOL
    wide = torch.randn(70, 333, generator=gen, device="cuda").half()
    out = torch.full((70, 401), 7.0, device="cuda", dtype=torch.bfloat16)
    _say("strided, off alignment, transposed, out=")
    for view in (wide[:, 1:130], wide[3:, 5:77], wide.t(), wide[::2], wide.t()[1:200, 3:50]):
        assert _far(orthogonalize(view), _exact(view)) <= TOL
    res = orthogonalize(wide[:, 2:302], out=out[:, 1:301])
    assert res.data_ptr() == out[:, 1:301].data_ptr() and _far(out[:, 1:301], _exact(wide[:, 2:302])) <= TOL
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 301:] == 7).all())


def test_scale_does_not_matter_and_spectra_of_any_kind(gpu):
    """Inputs from 1e-18 to 1e18 (fp32), low rank plus noise, rank one, one
    element, and an orthogonal matrix."""
    import torch
    from distributedspeed_amd import orthogonalize
    gen = _gen(5)
    base = _matrix(gen, 96, 200, torch.float32, std=1.0)
    for s in (1e-4, 1.0, 1e4, 1e18):
        _say(f"scale {s}")
        assert _far(orthogonalize(base * s), _exact(base * s)) <= TOL
    low = _matrix(gen, 256, 4, torch.float32, 1.0).mm(_matrix(gen, 4, 300, torch.float32, 1.0))
    spiked = low + _matrix(gen, 256, 300, torch.float32, 1.0)
    rank1 = _matrix(gen, 64, 1, torch.float32, 1.0).mm(_matrix(gen, 1, 64, torch.float32, 1.0))
    one = torch.zeros(48, 80, device="cuda")
    one[7, 9] = -3.0
    eye = torch.eye(130, device="cuda")
    for name, g in (("low rank and noise", spiked), ("rank one", rank1), ("one element", one), ("identity", eye)):
        _say(name)
        assert _far(orthogonalize(g), _exact(g)) <= TOL


def test_zero_nan_and_inf(gpu):
    import torch
    from distributedspeed_amd import orthogonalize
    z = torch.zeros(100, 37, device="cuda", dtype=torch.bfloat16)
    good = _matrix(_gen(6), 64, 64, torch.bfloat16)
    inf, nan = good.clone(), good.clone()
    inf[5, 6], nan[63, 0] = float("inf"), float("nan")
    _say("zero, inf, nan, good in one list")
    oz, oi, on, og = orthogonalize([z, inf, nan, good])
    assert bool((oz == 0).all())
    assert bool(oi.isnan().all()) and bool(on.isnan().all())
    assert _far(og, _exact(good)) <= TOL


def test_coefficients_of_each_step(gpu):
    import torch
    from distributedspeed_amd import orthogonalize
    g = _matrix(_gen(7), 80, 120, torch.float32)
    rows = ((4.0, -6.0, 2.8), (3.9, -5.9, 2.7), (2.5, -2.5, 1.0), (1.875, -1.25, 0.375))
    _say("four triples")
    got = orthogonalize(g, steps=4, coefficients=rows, eps=1e-6)
    assert _far(got, _exact(g, rows, 1e-6)) <= TOL
    one = orthogonalize(g, steps=1)
    assert _far(one, _exact(g, (COEF,))) <= TOL


def test_repeats_bit_for_bit_on_another_stream_and_in_a_graph(gpu):
    import torch
    from distributedspeed_amd import orthogonalize
    ms = [_matrix(_gen(8), 300, 520, torch.bfloat16), _matrix(_gen(9), 700, 96, torch.bfloat16)]
    first = orthogonalize(ms)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = orthogonalize(ms)
        outs = [torch.empty_like(o) for o in first]
        orthogonalize(ms, out=outs)
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, outs):
        assert torch.equal(a, b) and torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        orthogonalize(ms, out=outs)
    for k in range(3):
        _say(f"replay {k}")
        fresh = [_matrix(_gen(20 + k), *m.shape, torch.bfloat16) for m in ms]
        want = orthogonalize(fresh)
        for m, f in zip(ms, fresh):
            m.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_refusals(gpu):
    import torch
    from distributedspeed_amd import MuonOptimizer, orthogonalize
    g = torch.ones(4, 6, device="cuda")
    for bad, kind in (({"steps": 0}, ValueError), ({"steps": 65}, ValueError), ({"eps": 0.0}, ValueError),
                      ({"eps": float("nan")}, ValueError), ({"coefficients": (1.0, 2.0)}, ValueError),
                      ({"coefficients": ((1.0, 2.0, 3.0),) * 4}, ValueError),
                      ({"coefficients": (1.0, float("inf"), 0.0)}, ValueError),
                      ({"out": torch.empty(4, 6, device="cuda")}, ValueError),
                      ({"out": torch.empty(6, 4, device="cuda", dtype=torch.bfloat16).t()}, ValueError)):
        with pytest.raises(kind):
            orthogonalize(g, **bad)
    with pytest.raises(ValueError):
        orthogonalize(torch.ones(4, 6))
    with pytest.raises(ValueError):
        orthogonalize(torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        orthogonalize([g, torch.ones(3, device="cuda")])
    with pytest.raises(TypeError):
        orthogonalize([g, "x"])
    with pytest.raises(TypeError):
        orthogonalize([g, g.half()])
    with pytest.raises(TypeError):
        orthogonalize(g.double())
    assert orthogonalize([]) == []
    assert orthogonalize(torch.empty(0, 5, device="cuda")).shape == (0, 5)
    assert orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    p = torch.nn.Parameter(torch.ones(4, 4, device="cuda"))
    for bad in (dict(lr=-1.0), dict(weight_decay=-0.1), dict(momentum=1.0), dict(adjust_lr="x"), dict(ns_steps=0),
                dict(eps=0.0)):
        with pytest.raises(ValueError):
            MuonOptimizer([p], **bad)
    with pytest.raises(ValueError):
        MuonOptimizer([torch.nn.Parameter(torch.ones(4, device="cuda"))])
    with pytest.raises(ValueError):
        MuonOptimizer([torch.nn.Parameter(torch.ones(4, 6, device="cuda").t())])
    opt = MuonOptimizer([p])
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError):
        opt.step(grad_scale=2.0)
    with pytest.raises(ValueError):
        opt.step(grad_scale=torch.ones(2, device="cuda"))


# ---- the optimizer ------------------------------------------------------------------------------

def _muon_exact(w, buf, g, lr, wd, mu, nesterov, adjust):
    buf = mu * buf + (1 - mu) * g
    u = mu * buf + (1 - mu) * g if nesterov else buf
    rows, cols = w.shape
    f = 0.2 * math.sqrt(max(rows, cols)) if adjust == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))
    return w * (1 - lr * wd) - lr * f * _exact(u), buf, lr * f * math.sqrt(min(rows, cols))


@pytest.mark.parametrize("pdt,gdt", [("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "float32"),
                                     ("bfloat16", "float32")])
@pytest.mark.parametrize("nesterov,adjust", [(True, "original"), (False, "match_rms_adamw")])
def test_muon_steps(gpu, pdt, gdt, nesterov, adjust):
    """Three steps with a grad scale, over matrices of both orientations and
    odd sizes. The master is compared in units of one step's update norm: the
    bound of the iteration without the bf16 rounding, a step (15 * 2^-12), and
    fp32's rounding of the weights. The parameter is the master's cast."""
    import torch
    from distributedspeed_amd import MuonOptimizer
    pdt, gdt = getattr(torch, pdt), getattr(torch, gdt)
    gen = _gen(11)
    lr, wd, mu, scale = 0.02, 0.1, 0.95, 64.0
    ps = [torch.nn.Parameter(_matrix(gen, n, m, pdt, 0.05)) for n, m in ((64, 64), (100, 37), (37, 301), (260, 129))]
    opt = MuonOptimizer(ps, lr=lr, weight_decay=wd, momentum=mu, nesterov=nesterov, adjust_lr=adjust)
    ws, bufs = [p.detach().double() for p in ps], [torch.zeros(p.shape, device="cuda", dtype=torch.float64) for p in ps]
    gscale = torch.full((1,), scale, device="cuda")
    for step in range(3):
        _say(f"muon step {step}")
        units = []
        for k, p in enumerate(ps):
            g = _matrix(gen, *p.shape, torch.float32, 1e-2 * scale).to(gdt)
            p.grad = g if g.dtype == p.dtype else None
            if p.grad is None:
                p.grad_dtype = None
                p.grad = g
            ws[k], bufs[k], unit = _muon_exact(ws[k], bufs[k], g.double() / scale, lr, wd, mu, nesterov, adjust)
            units.append(unit)
        opt.step(grad_scale=gscale)
    assert not opt.last_step_skipped()
    for k, p in enumerate(ps):
        st = opt.state[p]
        master = st.get("master", p.detach())
        assert (master.double() - ws[k]).norm().item() <= 3 * 15 * 2.0 ** -12 * units[k] + 1e-6 * ws[k].norm().item()
        assert (st["momentum_buffer"].double() - bufs[k]).norm().item() <= 9 * 2.0 ** -23 * bufs[k].norm().item()
        assert torch.equal(p.detach(), master.to(pdt))


def test_muon_skips_on_overflow_and_restores_from_a_state_dict(gpu):
    import copy

    import torch
    from distributedspeed_amd import MuonOptimizer
    gen = _gen(12)

    def build():
        ps = [torch.nn.Parameter(_matrix(_gen(13), 50, 70, torch.bfloat16, 0.05)),
              torch.nn.Parameter(_matrix(_gen(14), 130, 40, torch.bfloat16, 0.05))]
        return ps, MuonOptimizer(ps, lr=0.02)

    ps, opt = build()
    grads = [[_matrix(gen, *p.shape, torch.bfloat16, 1e-2) for p in ps] for _ in range(3)]
    for p, g in zip(ps, grads[0]):
        p.grad = g.clone()
    opt.step()
    saved, weights = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in ps]
    before = [{k: v.clone() for k, v in opt.state[p].items()} for p in ps]
    ps[1].grad[3, 3] = float("nan")
    _say("a NaN in one grad")
    opt.step()
    assert opt.last_step_skipped()
    for p, w, b in zip(ps, weights, before):
        assert torch.equal(p.detach(), w) and all(torch.equal(opt.state[p][k], v) for k, v in b.items())
    for p, g in zip(ps, grads[1]):
        p.grad = g.clone()
    opt.step()
    assert not opt.last_step_skipped()
    others, opt2 = build()
    with torch.no_grad():
        for p, w in zip(others, weights):
            p.copy_(w)
    opt2.load_state_dict(saved)
    assert all(opt2.state[p]["master"].dtype == torch.float32 for p in others)
    for p, g in zip(others, grads[1]):
        p.grad = g.clone()
    opt2.step()
    for p, q in zip(ps, others):
        assert torch.equal(p.detach(), q.detach()) and torch.equal(opt.state[p]["master"], opt2.state[q]["master"])


def test_muon_takes_params_without_grads_and_strided_grads(gpu):
    import torch
    from distributedspeed_amd import MuonOptimizer
    a = torch.nn.Parameter(_matrix(_gen(15), 33, 65, torch.float32, 0.05))
    b = torch.nn.Parameter(_matrix(_gen(16), 20, 20, torch.float32, 0.05))
    opt = MuonOptimizer([a, b], lr=0.01, weight_decay=0.0)
    g = _matrix(_gen(17), 65, 33, torch.float32)
    a.grad = g.t()
    w, unchanged = a.detach().double(), b.detach().clone()
    want, _, unit = _muon_exact(w, torch.zeros_like(w), g.t().double(), 0.01, 0.0, 0.95, True, "original")
    opt.step()
    assert (a.detach().double() - want).norm().item() <= 15 * 2.0 ** -12 * unit + 1e-6 * w.norm().item()
    assert torch.equal(b.detach(), unchanged) and not opt.state.get(b)
