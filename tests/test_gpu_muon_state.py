"""MuonOptimizer steps after its state or its parameters changed their type,
on the GPU against the step in 64 bits. Tolerance of a step: 15 roundings of
2^-12 in the iteration, in units of the update's norm, and fp32's rounding of
the weights (as for steps of one type)."""
from __future__ import annotations

import copy
import math
import sys

import pytest

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
SHAPES = ((70, 50), (33, 129), (40, 40))


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _exact(g):
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        p = x.mm(x.t().contiguous())
        x = COEF[0] * x + (COEF[1] * p + COEF[2] * p.mm(p)).mm(x)
    return x.t() if tall else x


def _normal(gen, shape, std):
    import torch
    return torch.randn(shape, generator=gen, device="cuda") * std


def _build(dtype, seed):
    import torch
    from distributedspeed_amd import MuonOptimizer
    gen = torch.Generator("cuda").manual_seed(seed)
    ps = [torch.nn.Parameter(_normal(gen, s, 0.05).to(getattr(torch, dtype))) for s in SHAPES]
    return ps, MuonOptimizer(ps, lr=0.02, weight_decay=0.1), gen


def _grads(ps, gen):
    for p in ps:
        p.grad = _normal(gen, p.shape, 1e-2).to(p.dtype)


def _weights(opt, p):
    return opt.state[p].get("master", p.detach()).double()


def _step_and_check(opt, ps, weights, buffers):
    """One step from the given fp64 weights and momenta."""
    opt.step()
    assert not opt.last_step_skipped()
    for p, w, buf in zip(ps, weights, buffers):
        g = p.grad.double()
        buf = 0.95 * buf + 0.05 * g
        factor = 0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        want = w * (1 - 0.02 * 0.1) - factor * _exact(0.95 * buf + 0.05 * g)
        unit = factor * math.sqrt(min(p.shape))
        assert (_weights(opt, p) - want).norm().item() <= 15 * 2.0 ** -12 * unit + 1e-6 * w.norm().item()
        got = opt.state[p]["momentum_buffer"].double()
        assert (got - buf).norm().item() <= 3 * 2.0 ** -23 * buf.norm().item()


@pytest.mark.parametrize("saved", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_state_of_one_type_into_parameters_of_another(gpu, saved, dtype):
    ps, opt, gen = _build(saved, 1)
    _grads(ps, gen)
    opt.step()
    qs, other, gen2 = _build(dtype, 2)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    _grads(qs, gen2)
    _say(f"state of {saved} into {dtype}")
    weights = [q.detach().double() if saved == "float32" else _weights(opt, p) for p, q in zip(ps, qs)]
    _step_and_check(other, qs, weights, [opt.state[p]["momentum_buffer"].double() for p in ps])


@pytest.mark.parametrize("before,after", [("float32", "bfloat16"), ("bfloat16", "float32"), ("float16", "bfloat16")])
def test_parameters_cast_between_steps(gpu, before, after):
    import torch
    ps, opt, gen = _build(before, 3)
    _grads(ps, gen)
    opt.step()
    kept = [_weights(opt, p) for p in ps]
    for p in ps:
        p.grad = None
        p.data = p.data.to(getattr(torch, after))
    weights = [p.detach().double() for p in ps] if before == "float32" else kept
    _grads(ps, gen)
    _say(f"{before} cast to {after}")
    _step_and_check(opt, ps, weights, [opt.state[p]["momentum_buffer"].double() for p in ps])


@pytest.mark.parametrize("adjust", [None, "match_rms_adamw"])
def test_goes_on_from_torchs_muon(gpu, adjust):
    """torch.optim.Muon's state dict, then one step of each from there. Torch
    rounds its input and three products a step to bf16 (2^-9 each): 16
    roundings of 2^-9 beside this class's own."""
    import torch
    from distributedspeed_amd import MuonOptimizer
    gen = torch.Generator("cuda").manual_seed(4)
    ps = [torch.nn.Parameter(_normal(gen, s, 0.05)) for s in SHAPES]
    theirs = torch.optim.Muon(ps, lr=0.02, weight_decay=0.1, adjust_lr_fn=adjust)
    _grads(ps, gen)
    theirs.step()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = MuonOptimizer(qs)
    opt.load_state_dict(copy.deepcopy(theirs.state_dict()))
    _grads(ps, gen)
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    _say(f"one step of each, adjust_lr_fn={adjust}")
    theirs.step()
    opt.step()
    for p, q in zip(ps, qs):
        factor = 0.2 * math.sqrt(max(p.shape)) if adjust else math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        unit = 0.02 * factor * math.sqrt(min(p.shape))
        far = (p.detach().double() - q.detach().double()).norm().item()
        assert far <= (16 * 2.0 ** -9 + 15 * 2.0 ** -12) * unit + 1e-6 * p.detach().norm().item(), far / unit


def test_a_dynamic_scale_shared_with_adamw(gpu):
    """The loop that MuonOptimizer's documentation gives, in fp16: the matrix's
    scaled grad overflows above 2^14, the vector's never. The scale comes down
    until Muon steps, both optimizers step together, and the scale's growth
    (after two clean steps) costs a skipped step, not the run."""
    import torch
    from distributedspeed_amd import AdamWOptimizer, MuonOptimizer
    from distributedspeed_amd.flat_step import ScalerConfig
    w = torch.nn.Parameter(_normal(torch.Generator("cuda").manual_seed(5), (40, 24), 0.05).half())
    v = torch.nn.Parameter(torch.full((64,), 0.5, device="cuda", dtype=torch.float16))
    muon = MuonOptimizer([w], lr=0.01)
    adamw = AdamWOptimizer([v], lr=1e-3, param_dtype=torch.float16,
                           loss_scaler=ScalerConfig(mode="dynamic", init_scale=2.0 ** 18, window=2, hysteresis=1))
    true = torch.full((40, 24), 0.5, device="cuda")
    true[3, 4] = 3.0  # times 2^14 below 65504, times 2^15 above
    seen = []
    for step in range(12):
        scale = adamw.loss_scale_tensor()
        w.grad = (true * scale).half()
        v.grad = None
        (v.float().sum() * 0.01 * scale).backward()
        before = [p.detach().clone() for p in (w, v)]
        muon.step(grad_scale=scale)
        used, skipped = float(scale), muon.last_step_skipped()
        if skipped:
            adamw.set_scaler_state(adamw.read_state().scale / 2)
        else:
            adamw.step()
        _say(f"step {step}: scale 2^{math.log2(used):g}, skipped {skipped}")
        assert skipped == (used > 2.0 ** 14)
        for p, old in zip((w, v), before):
            assert torch.equal(p.detach(), old) == skipped
        seen.append(skipped)
    # 2^18 to 2^15 skipped; then two steps, growth, one skipped
    assert seen == [True] * 4 + [False, False, True, False, False, True, False, False]
