"""The sequence operators as a training program meets them: a small language model
of them and of the feed-forward blocks against plain 64-bit layers, under the
engine, from several streams and threads, captured forwards, and the example.

Tolerance of the model's gradients, of the Frobenius norm: some 25 roundings of the
type lie between a parameter and its gradient, forward and backward, each of 2^-9
(bf16, root mean square); were they all to point the same way, 25 * 2^-9 = 4.9%."""
from __future__ import annotations

import math
import os
import sys
import threading

import pytest

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _example():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    try:
        import train_packed_lm
    finally:
        sys.path.pop(0)
    return train_packed_lm


def _plain_loss(p, blocks, tokens, targets, lengths, heads, kv_heads):
    """The model in 64 bits, sequence by sequence where it matters."""
    import torch
    F = torch.nn.functional

    def rms(v, w):
        return v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w

    def turned(x, at):
        half = x.shape[-1] // 2
        angle = at.double()[:, None, None] * 10000.0 ** (-torch.arange(half, device=x.device).double() / half)
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

    def attention(q, k, v):
        out, first = [], 0
        for n in lengths:
            at = slice(first, first + n)
            first += n
            where = torch.arange(n, device=q.device)
            a, b = turned(q[at], where), turned(k[at], where).repeat_interleave(heads // kv_heads, 1)
            c = v[at].repeat_interleave(heads // kv_heads, 1)
            s = torch.einsum("ihd,jhd->hij", a, b) / math.sqrt(q.shape[-1])
            s = s.masked_fill(where[:, None] < where, -math.inf)
            out.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), c))
        return torch.cat(out)

    h = F.embedding(tokens, p["embedding"])
    normed = rms(h, p["first_weight"])
    for i in range(blocks):
        a = {n: p[f"attention.{i}.{n}"] for n in ("w_q", "w_k", "w_v", "w_o", "post_weight", "gate", "next_weight")}
        rows = normed.shape[0]
        q, k, v = (F.linear(normed, a[n]).view(rows, c, -1) for n, c in (("w_q", heads), ("w_k", kv_heads), ("w_v", kv_heads)))
        y = F.linear(attention(q, k, v).reshape(rows, -1), a["w_o"])
        h = h + a["gate"] * rms(y, a["post_weight"])
        normed = rms(h, a["next_weight"])
        f = {n: p[f"ffn.{i}.{n}"] for n in ("w_gate", "w_up", "w_down", "post_weight", "gate", "next_weight")}
        y = F.linear(F.silu(F.linear(normed, f["w_gate"])) * F.linear(normed, f["w_up"]), f["w_down"])
        h = h + f["gate"] * rms(y, f["post_weight"])
        normed = rms(h, f["next_weight"])
    return F.cross_entropy(F.linear(normed, p["embedding"]), targets, ignore_index=-100)


def test_a_language_model_of_them(gpu):
    import torch
    from distributedspeed_amd import PackedSequences
    lm = _example()
    torch.manual_seed(0)
    model = lm.PackedLM(300, 96, 4, 2, 2, device="cuda", dtype=torch.bfloat16)
    tokens, targets, lengths = lm.batch(300, 700, torch.Generator().manual_seed(1))
    tokens, targets = tokens.cuda(), targets.cuda()
    _say(f"a model over sequences of {lengths}")
    loss = model(tokens, targets, PackedSequences(lengths))
    loss.backward()
    p = {n: t.detach().double().requires_grad_(True) for n, t in model.named_parameters()}
    want = _plain_loss(p, 2, tokens, targets, lengths, 4, 2)
    grads = torch.autograd.grad(want, list(p.values()))
    assert abs(loss.item() - want.item()) <= 0.02 * want.item()
    for (name, t), g in zip(model.named_parameters(), grads):
        far = ((t.grad.double() - g).norm() / g.norm()).item()
        assert far <= 25 * 2.0 ** -9, (name, far)


@pytest.mark.parametrize("precision", ["bf16", "fp16"])
def test_under_the_engine(gpu, precision):
    """Parameters at any element's address of one 16-bit buffer, cast inputs, loss
    scaling: the first gradients are the model's own on the cast parameters, and
    every step's loss is finite."""
    import torch
    import distributedspeed_amd as ds
    from distributedspeed_amd import PackedSequences
    lm = _example()

    class Model(torch.nn.Module):
        def __init__(self, **kw):
            super().__init__()
            self.odd = torch.nn.Parameter(torch.ones(3, **kw))  # what lies behind it is off 16 bytes
            self.lm = lm.PackedLM(200, 64, 4, 2, 1, **kw)

        def forward(self, tokens, targets, packing):
            return self.lm(tokens, targets, packing) * self.odd.float().mean()

    torch.manual_seed(0)
    model = Model()
    initial = {n: p.detach().clone() for n, p in model.named_parameters()}
    scaling = {"loss_scale": 0, "initial_scale_power": 8} if precision == "fp16" else {}
    engine, _, _, _ = ds.initialize(model, {precision: {"enabled": True, **scaling},
                                            "optimizer": {"type": "AdamW", "params": {"lr": 3e-3}}})
    dt = torch.bfloat16 if precision == "bf16" else torch.float16
    other = Model(device="cuda", dtype=dt)
    with torch.no_grad():
        for n, p in other.named_parameters():
            p.copy_(initial[n])
    gen = torch.Generator().manual_seed(2)
    for step in range(6):
        tokens, targets, lengths = lm.batch(200, 300, gen)
        packing = PackedSequences(lengths)
        loss = engine(tokens.cuda(), targets.cuda(), packing)
        if step == 0:
            ref = other(tokens.cuda(), targets.cuda(), packing)
            assert abs(loss.item() - ref.item()) <= 1e-2 * ref.item()
            want = torch.autograd.grad(ref, list(other.parameters()))
            got = torch.autograd.grad(engine.module(tokens.cuda(), targets.cuda(), packing), list(engine.module.parameters()))
            for (n, p), a, b in zip(other.named_parameters(), got, want):
                assert (a.float() - b.float()).norm() <= 25 * 2.0 ** -9 * b.float().norm(), n
        engine.backward(loss)
        engine.step()
        _say(f"{precision}: step {step} loss {loss.item():.4f}")
        assert math.isfinite(loss.item())


def test_the_block_is_its_operators(gpu):
    """Padded rows behind the sequences, which hold anything, change nothing."""
    import torch
    from distributedspeed_amd import AttentionBlock, PackedSequences, gated_residual_norm, packed_attention, rotary
    torch.manual_seed(1)
    b = AttentionBlock(96, 4, 2, 32, gate_init=0.5, branch_scale=0.7, rotary_base=5e4, device="cuda", dtype=torch.bfloat16)
    packing = PackedSequences([33, 0, 90, 1])
    assert packing.offsets.tolist() == [0, 33, 33, 123, 124] and packing.tokens == 124
    assert packing.positions.tolist() == list(range(33)) + list(range(90)) + [0]
    x = torch.randn(124, 96, device="cuda").bfloat16()
    h, n = b(x, x, packing)
    linear = torch.nn.functional.linear
    q, k, v = linear(x, b.w_q).view(124, 4, 32), linear(x, b.w_k).view(124, 2, 32), linear(x, b.w_v).view(124, 2, 32)
    q, k = rotary(q, k, packing.positions, base=5e4)
    y = linear(packed_attention(q, k, v, packing).reshape(124, 128), b.w_o)
    h2, n2 = gated_residual_norm(x, y, post_weight=b.post_weight, gate=b.gate, next_weight=b.next_weight, branch_scale=0.7)
    assert torch.equal(h, h2) and torch.equal(n, n2)
    more = torch.cat((x, torch.full((6, 96), 7.0, device="cuda").bfloat16()))
    h3, n3 = b(more, more, packing)
    # (the library's products may add in another order for another number of rows)
    assert h3.shape == (130, 96) and ((h3[:124] - h).float().norm() <= 2.0 ** -7 * h.float().norm())
    assert n3.isfinite().all()


def _work(seed):
    """A call of each operator with gradients; fresh leaves."""
    import torch
    from distributedspeed_amd import PackedSequences, linear_cross_entropy, packed_attention, rotary
    gen = torch.Generator("cuda").manual_seed(seed)
    rows = torch.randn(300, 6, 64, generator=gen, device="cuda").bfloat16()
    q, k, v = (rows[:, a:b].detach().clone().requires_grad_(True) for a, b in ((0, 4), (4, 5), (5, 6)))
    w = (torch.randn(500, 256, generator=gen, device="cuda") / 16).bfloat16().requires_grad_(True)
    targets = torch.randint(0, 500, (300,), generator=gen, device="cuda")
    packing = PackedSequences([100, 150, 50])

    def run():
        a, b = rotary(q, k, packing.positions)
        loss = linear_cross_entropy(packed_attention(a, b, v, packing).view(300, 256), w, targets)
        return [loss.detach(), *torch.autograd.grad(loss, [q, k, v, w])]

    return run


def test_other_streams_and_threads(gpu):
    """Side by side on two streams from two threads, many calls at once in flight:
    to the bit what one stream gives."""
    import torch
    works = [_work(s) for s in range(2)]
    want = [w() for w in works]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def go(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i].append(works[i]())
            stream.synchronize()
        except Exception as e:  # noqa: BLE001  (shown below)
            errors.append(e)

    threads = [threading.Thread(target=go, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_captured_forwards(gpu):
    """Replayed with other inputs in place, eager work and synchronisations between,
    two graphs of one memory pool in turn."""
    import torch
    from distributedspeed_amd import PackedSequences, linear_cross_entropy, packed_attention, rotary
    packing = PackedSequences([130, 70, 1])
    positions = packing.positions
    gen = torch.Generator("cuda").manual_seed(0)

    def fresh():
        return (torch.randn(201, 6, 64, generator=gen, device="cuda").bfloat16(),
                torch.randint(-1, 300, (201,), generator=gen, device="cuda"))

    w = (torch.randn(300, 256, generator=gen, device="cuda") / 16).bfloat16()
    rows, targets = fresh()

    def run(rows, targets, reduction):
        q, k = rotary(rows[:, :4], rows[:, 4:5], positions)
        x = packed_attention(q, k, rows[:, 5:], packing)
        return x, linear_cross_entropy(x.view(201, 256), w, targets, ignore_index=-1, reduction=reduction)

    with torch.no_grad():
        run(rows, targets, "mean")
        graphs = []
        for reduction in ("mean", "none"):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
                out = run(rows, targets, reduction)
            graphs.append((g, out, reduction))
        for k in range(4):
            a, b = fresh()
            rows.copy_(a)
            targets.copy_(b)
            for g, out, reduction in graphs:
                want = run(a, b, reduction)
                g.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(x, y) for x, y in zip(out, want)), (k, reduction)


def test_a_captured_backward_is_refused(gpu):
    """Of each operator, with a message; the stream works on afterwards."""
    import torch
    from distributedspeed_amd import PackedSequences, linear_cross_entropy, packed_attention, rotary
    packing = PackedSequences([5, 3])
    x = torch.randn(8, 2, 64, device="cuda").bfloat16().requires_grad_(True)
    at = torch.zeros(8, dtype=torch.int64, device="cuda")
    for call in (lambda: packed_attention(x, x, x, packing), lambda: rotary(x, x, packing.positions)[0],
                 lambda: linear_cross_entropy(x.view(8, 128), x.view(8, 128), at)):
        out = call()
        dout = torch.ones_like(out)
        want = torch.autograd.grad(out, x, dout, retain_graph=True)[0]
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            out = call()
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream), pytest.raises(RuntimeError, match="captured"):
                torch.autograd.grad(out, x, dout)
            assert torch.equal(torch.autograd.grad(call(), x, dout)[0], want)


def test_the_example_trains(gpu):
    """It runs and every step's loss is finite."""
    losses = _example().train(256, 96, 4, 2, 2, 512, 8)
    _say(f"example: loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    assert len(losses) == 8 and all(math.isfinite(v) for v in losses)


def test_refusals(gpu):
    import torch
    from distributedspeed_amd import PackedSequences, linear_cross_entropy, packed_attention, rotary
    q, k = torch.zeros(10, 4, 16, device="cuda").bfloat16(), torch.zeros(10, 2, 16, device="cuda").bfloat16()
    p = PackedSequences([6, 4])
    wide = torch.zeros(10, 1, 257, device="cuda").bfloat16()
    for args, kw, kind in (((q, k, k, [6, 4]), {}, TypeError), ((q, k, k[:9], p), {}, ValueError),
                           ((q, k, k[:, :1], p), {}, ValueError), ((q[:, :3], k, k, p), {}, ValueError),
                           ((q[:8], k[:8], k[:8], p), {}, ValueError), ((q.half(), k, k, p), {}, TypeError),
                           ((q.float(), k.float(), k.float(), p), {}, TypeError), ((q, k.cpu(), k, p), {}, ValueError),
                           ((q.cpu(), k, k, p), {}, ValueError), ((q, None, k, p), {}, TypeError),
                           ((q[:, :0], k, k, p), {}, ValueError), ((q, k[:, :0], k[:, :0], p), {}, ValueError),
                           ((wide, wide, wide, p), {}, ValueError), ((q[..., :0], k[..., :0], k[..., :0], p), {}, ValueError),
                           ((q[0], k[0], k[0], p), {}, ValueError), ((q, k, k, p), dict(scale=0.0), ValueError),
                           ((q, k, k, p), dict(scale=float("nan")), ValueError)):
        with pytest.raises(kind):
            packed_attention(*args, **kw)
    at = torch.arange(10, device="cuda")
    for args, kw, kind in (((q, k, at.float()), {}, TypeError), ((q, k, at[:9]), {}, ValueError),
                           ((q, k[:9], at), {}, ValueError), ((q, k.half(), at), {}, TypeError),
                           ((q, k, at.cpu()), {}, ValueError), ((q[0], k[0], at[0]), {}, ValueError),
                           ((q.double(), k.double(), at), {}, TypeError), ((q, k, at), dict(dims=5), ValueError),
                           ((q, k, at), dict(dims=18), ValueError), ((q, k, at), dict(base=0.0), ValueError),
                           ((q, k, at), dict(base=float("inf")), ValueError), ((q, k[..., :8], at), {}, ValueError),
                           ((q, k, None), {}, TypeError)):
        with pytest.raises(kind):
            rotary(*args, **kw)
    x, w = q.view(10, 64), torch.zeros(30, 64, device="cuda").bfloat16()
    for args, kw, kind in (((x, w, at.float()), {}, TypeError), ((x, w, at[:9]), {}, ValueError),
                           ((x, w[:, :32], at), {}, ValueError), ((x, w.half(), at), {}, TypeError),
                           ((x.float(), w.float(), at), {}, TypeError), ((x, w, at.cpu()), {}, ValueError),
                           ((x, w[:0], at), {}, ValueError), ((x[:, :0], w[:, :0], at), {}, ValueError),
                           ((x, w, at), dict(reduction="max"), ValueError), ((x, None, at), {}, TypeError),
                           ((x, w, at), dict(ignore_index=2 ** 70), ValueError), ((x, w[0], at), {}, ValueError)):
        with pytest.raises(kind):
            linear_cross_entropy(*args, **kw)
