"""The autograd nodes of the sequence operators on CPU tensors, with stubs in the
place of the library: what they refuse before anything is called, what they hand
on, and which tensors they copy first."""
from __future__ import annotations

import ctypes

import pytest


@pytest.fixture()
def nodes():
    """The built module bound to stubs that write nothing and note what they are
    given. The next user of sequence.py binds the library again."""
    import torch  # noqa: F401  (the module links against it)
    from distributedspeed_amd import _lib, sequence
    from distributedspeed_amd import _sequence_autograd as m
    P, I64, I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    m.seen, m.capturing = {}, 0

    def note(name, struct):
        def f(q, *rest):
            m.seen[name] = (struct.from_buffer_copy((ctypes.c_char * ctypes.sizeof(struct)).from_address(q)), rest)
            return 0
        return f

    A, R, Z = _lib.DsxAttention, _lib.DsxRotary, _lib.DsxLoss
    m.stubs = {
        "dsx_last_error": ctypes.CFUNCTYPE(ctypes.c_char_p)(lambda: b""),
        "dsx_stream_capturing": ctypes.CFUNCTYPE(I32, P)(lambda s: m.capturing),
        "dsx_attention_forward": ctypes.CFUNCTYPE(I32, P, P, P, P, P)(note("attention", A)),
        "dsx_attention_workspace_bytes": ctypes.CFUNCTYPE(I64, P)(lambda *a: 256),
        "dsx_attention_backward": ctypes.CFUNCTYPE(I32, P, P, P, P, P, I64, I64, P, P, P, P, I64, P)(note("d_attention", A)),
        "dsx_rotary": ctypes.CFUNCTYPE(I32, P, P, P, I32, P)(note("rotary", R)),
        "dsx_loss_saved_bytes": ctypes.CFUNCTYPE(I64, P)(lambda *a: 256),
        "dsx_loss_workspace_bytes": ctypes.CFUNCTYPE(I64, P, I32)(lambda *a: 256),
        "dsx_loss_forward": ctypes.CFUNCTYPE(I32, P, P, P)(note("loss", Z)),
        "dsx_loss_backward": ctypes.CFUNCTYPE(I32, P, P, P, P, P)(note("d_loss", Z)),
    }
    m.bind({n: ctypes.cast(f, P).value for n, f in m.stubs.items()})
    yield m
    sequence._nodes = None


def _attention(nodes, q, k, v):
    import torch
    return nodes.packed_attention(q, k, v, torch.zeros(2, 1, 4, dtype=torch.int32), 10, 7, 58, True, 0.5, 0)


def _rotary(nodes, q, k):
    import torch
    return nodes.rotary(q, k, torch.arange(q.shape[0]), 1e4, q.shape[2] // 2 * 2, False, 0)


def _loss(nodes, x, w):
    import torch
    return nodes.linear_cross_entropy(x, w, torch.zeros(x.shape[0], dtype=torch.long), -100, 1, 0)


def _qkv(d=16, rows=12):
    import torch
    return [torch.ones(rows, h, d).bfloat16() for h in (4, 2, 2)]


def _calls(nodes):
    import torch
    return ((lambda: _qkv(), lambda a: _attention(nodes, *a)), (lambda: _qkv()[:2], lambda a: _rotary(nodes, *a)),
            (lambda: [torch.ones(4, 8).bfloat16(), torch.ones(30, 8).bfloat16()], lambda a: _loss(nodes, *a)))


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("tracked", [False, True])
def test_a_forward_mode_tangent_is_refused(nodes, tracked, no_grad):
    import torch
    import torch.autograd.forward_ad as fw
    for make, call in _calls(nodes):
        for k in range(len(make())):
            args = make()
            if tracked:
                args[-1].requires_grad_(True)
            with fw.dual_level(), torch.set_grad_enabled(not no_grad):
                args[k] = fw.make_dual(args[k], torch.ones_like(args[k]))
                with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                    call(args)


def test_a_captured_backward_is_refused(nodes):
    for make, call in _calls(nodes):
        args = [t.requires_grad_(True) for t in make()]
        out = call(args)
        out = out[0] if isinstance(out, tuple) else out
        nodes.capturing = 1
        with pytest.raises(RuntimeError, match="captured"):
            out.float().sum().backward()
        nodes.capturing = 0


def test_differentiable_once(nodes):
    import torch
    for make, call in _calls(nodes):
        args = [t.requires_grad_(True) for t in make()]
        out = call(args)
        out = out[0] if isinstance(out, tuple) else out
        g, = torch.autograd.grad(out, args[0], torch.ones_like(out).requires_grad_(True), create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            g.float().sum().backward()


def test_attention_hands_on_strides_and_copies_what_it_must(nodes):
    import torch
    rows = torch.ones(12, 8, 16).bfloat16()
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    out = _attention(nodes, q, k, v)
    a = nodes.seen["attention"][0]
    assert (a.ld_q, a.head_q, a.ld_k, a.tokens, a.longest, a.pairs) == (128, 16, 128, 10, 7, 58)
    assert (a.heads, a.kv_heads, a.head_dim) == (4, 2, 16)
    assert a.q == q.data_ptr() and a.k == k.data_ptr() and a.v == v.data_ptr()
    assert out.shape == (12, 4, 16) and not out[10:].any()  # rows behind the sequences
    for bad in (torch.ones(12, 4, 32).bfloat16()[..., ::2], torch.ones(12, 4, 15).bfloat16(),
                torch.ones(12 * 64 + 1).bfloat16()[1:].view(12, 4, 16), torch.ones(12, 1, 16).bfloat16().expand(-1, 4, -1),
                torch.ones(1, 4, 16).bfloat16().expand(12, -1, -1), torch.ones(12, 68).bfloat16()[:, :64].view(12, 4, 16)):
        d = bad.shape[2]
        kv = torch.ones(12, 2, d).bfloat16()
        out = _attention(nodes, bad, kv, kv)
        a = nodes.seen["attention"][0]
        assert a.q != bad.data_ptr() and a.ld_q % 8 == 0 and a.head_q >= a.head_dim == -(-d // 8) * 8
        assert out.shape == (12, 4, d)


def test_backward_computes_what_is_wanted(nodes):
    import torch
    for wanted in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        args = [t.requires_grad_(bool(w)) for t, w in zip(_qkv(d=12), wanted)]
        _attention(nodes, *args).float().sum().backward()
        _, rest = nodes.seen["d_attention"]
        dq, dk, dv = rest[6:9]
        assert bool(dq) == bool(wanted[0]) and bool(dk) == bool(dv) == bool(wanted[1] or wanted[2])
        for t, w in zip(args, wanted):
            assert (t.grad is not None) == bool(w) and (not w or (t.grad.shape == t.shape and not t.grad[10:].any()))
    x, w = torch.ones(4, 8).bfloat16(), torch.ones(30, 8).bfloat16().requires_grad_(True)
    _loss(nodes, x, w).backward()
    assert not nodes.seen["d_loss"][1][1] and nodes.seen["d_loss"][1][2] and w.grad.shape == w.shape


def test_rotary_with_one_gradient(nodes):
    q, k = (t.requires_grad_(True) for t in _qkv()[:2])
    y, z = _rotary(nodes, q, k)
    z.float().sum().backward()
    a = nodes.seen["rotary"][0]
    assert (a.heads, a.kv_heads) == (2, 0) and nodes.seen["rotary"][1][2] == 1  # k's alone, turned back
    assert k.grad.shape == k.shape
