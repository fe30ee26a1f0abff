"""The block operators as a training program meets them: the gradients beside a
non-finite token, and GatedFFNBlock under the engine.

Tolerance of a gradient: three roundings of the type (2^-9 for bf16, root mean
square), of the Frobenius norm."""
from __future__ import annotations

import sys

import pytest

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("tokens,d,f", [(3, 72, 200), (40, 520, 136), (200, 100, 300), (300, 512, 1024)])
def test_gradients_beside_a_non_finite_token(gpu, tokens, d, f, value):
    """dx of every other token is what it is without that one, to the bit, and
    as close to 64 bits as ever; its own row and the weights' gradients, which
    it is a term of, are not finite."""
    import torch
    from distributedspeed_amd import gated_ffn
    gen = torch.Generator("cuda").manual_seed(tokens)

    def normal(*s, std=1.0):
        return (torch.randn(*s, generator=gen, device="cuda") * std).bfloat16()

    x, wg, wu, wd = normal(tokens, d), normal(f, d, std=d ** -0.5), normal(f, d, std=d ** -0.5), normal(d, f, std=f ** -0.5)
    dy = normal(tokens, d, std=0.1)

    def grads(x):
        args = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
        return torch.autograd.grad(gated_ffn(*args), args, dy)

    clean = grads(x)
    bad = x.clone()
    bad[1, d - 1] = value
    _say(f"{value} in one of {tokens} tokens of {d} x {f}")
    got = grads(bad)
    keep = [i for i in range(tokens) if i != 1]
    assert torch.equal(got[0][keep], clean[0][keep])
    assert not bool(got[0][1].isfinite().all())
    assert all(not bool(g.isfinite().all()) for g in got[1:])
    args = [t.double().requires_grad_(True) for t in (x, wg, wu, wd)]
    F = torch.nn.functional
    y = F.linear(F.silu(F.linear(args[0], args[1])) * F.linear(args[0], args[2]), args[3])
    want, = torch.autograd.grad(y, args[0], dy.double())
    assert (got[0][keep].double() - want[keep]).norm() <= 3 * 2.0 ** -9 * want[keep].norm()


@pytest.mark.parametrize("width,inner", [(64, 176), (48, 100)])
@pytest.mark.parametrize("precision", ["bf16", "fp16"])
def test_the_block_under_the_engine(gpu, precision, width, inner):
    """Blocks built in fp32 and given to initialize(), which re-homes their
    parameters into one 16-bit buffer (at any element's address) and casts the
    inputs: the first forward and gradients are the operators' own on the cast
    parameters (another load path where addresses differ, so within the ten or
    so roundings of 2^-9 that the blocks make), and the loss falls."""
    import torch
    import distributedspeed_amd as ds
    from distributedspeed_amd import GatedFFNBlock, gated_residual_norm

    class Stack(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.first_weight = torch.nn.Parameter(torch.ones(width))
            self.odd = torch.nn.Parameter(torch.ones(3))  # the matrices behind it lie off 16 bytes
            self.blocks = torch.nn.ModuleList(GatedFFNBlock(width, inner, gate_init=0.5) for _ in range(2))

        def forward(self, x):
            hidden, normed = gated_residual_norm(x, next_weight=self.first_weight)
            for block in self.blocks:
                hidden, normed = block(hidden, normed)
            return normed * self.odd.mean()

    torch.manual_seed(0)
    model = Stack()
    initial = {n: p.detach().clone() for n, p in model.named_parameters()}
    scaling = {"loss_scale": 0, "initial_scale_power": 8} if precision == "fp16" else {}
    engine, _, _, _ = ds.initialize(model, {precision: {"enabled": True, **scaling}, "optimizer": {"type": "AdamW", "params": {"lr": 3e-3}}})
    dt = torch.bfloat16 if precision == "bf16" else torch.float16
    other = Stack().cuda().to(dt)
    with torch.no_grad():
        for n, p in other.named_parameters():
            p.copy_(initial[n])
    target = torch.randn(width, width, device="cuda") / width ** 0.5
    losses = []
    for step in range(40):
        x = torch.randn(96, width, device="cuda")
        want = torch.tanh(x.to(dt).float() @ target)
        loss = (engine(x).float() - want).square().mean()
        if step == 0:
            _say(f"{precision}: the first step's gradients")
            ref = (other(x.to(dt)).float() - want).square().mean()
            assert abs(loss.item() - ref.item()) <= 1e-2 * ref.item()
            names, params = zip(*other.named_parameters())
            grads = dict(zip(names, torch.autograd.grad(ref * 256.0, params)))
        engine.backward(loss)
        if step == 0:
            scale = engine.loss_scale
            for n, p in engine.module.named_parameters():
                g = grads[n].double() / 256.0
                assert (p.grad.double() / scale - g).norm() <= 0.05 * g.norm() + 1e-7, n
        engine.step()
        losses.append(loss.item())
    _say(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5])
