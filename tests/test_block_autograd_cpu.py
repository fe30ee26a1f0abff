"""The autograd nodes of the block operators on CPU tensors, with stubs in the
place of the library: what they refuse before anything is called."""
from __future__ import annotations

import ctypes

import pytest


@pytest.fixture()
def nodes():
    """The built module bound to stubs that write nothing. The next user of
    block.py binds the library again."""
    import torch  # noqa: F401  (the module links against it)
    from distributedspeed_amd import _block_autograd as m
    from distributedspeed_amd import block
    P, I64, I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    stubs = {
        "dsx_last_error": ctypes.CFUNCTYPE(ctypes.c_char_p)(lambda: b""),
        "dsx_ffn_saved_bytes": ctypes.CFUNCTYPE(I64, I64, I64, I32)(lambda *a: 256),
        "dsx_ffn_workspace_bytes": ctypes.CFUNCTYPE(I64, P, I32)(lambda *a: 256),
        "dsx_ffn_forward": ctypes.CFUNCTYPE(I32, P, P, I64, P)(lambda *a: 0),
        "dsx_ffn_backward": ctypes.CFUNCTYPE(I32, P, P, I64, P, I64, P, P, P, P)(lambda *a: 0),
        "dsx_norm_workspace_bytes": ctypes.CFUNCTYPE(I64, P)(lambda *a: 256),
        "dsx_norm_forward": ctypes.CFUNCTYPE(I32, P, P, P, P)(lambda *a: 0),
        "dsx_norm_backward": ctypes.CFUNCTYPE(I32, P, P, I64, P, I64, P, P, P, P, P, P, I64, P)(lambda *a: 0),
    }
    m.bind({n: ctypes.cast(f, P).value for n, f in stubs.items()})
    yield m
    block._nodes = None


def _ffn():
    import torch
    return [torch.ones(4, 8).bfloat16(), torch.ones(16, 8).bfloat16(), torch.ones(16, 8).bfloat16(),
            torch.ones(8, 16).bfloat16()]


def _norm():
    import torch
    return [torch.ones(4, 8), torch.ones(4, 8), torch.ones(8), torch.ones(8), torch.ones(8)]


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("tracked", [False, True])
def test_a_forward_mode_tangent_is_refused(nodes, tracked, no_grad):
    """In any input, whether or not an input requires grad."""
    import torch
    import torch.autograd.forward_ad as fw
    for make, call in ((_ffn, lambda a: nodes.gated_ffn(*a, 0, 0)),
                       (_norm, lambda a: nodes.gated_residual_norm(*a, 1.0, 1.0, 1e-6, 0))):
        for k in range(len(make())):
            args = make()
            if tracked:
                args[-1].requires_grad_(True)
            with fw.dual_level(), torch.set_grad_enabled(not no_grad):
                args[k] = fw.make_dual(args[k], torch.ones_like(args[k]))
                with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                    call(args)


def test_plain_inputs_are_taken(nodes):
    import torch
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        assert nodes.gated_ffn(*_ffn(), 0, 0).shape == (4, 8)
        hidden, normed = nodes.gated_residual_norm(*_norm(), 1.0, 1.0, 1e-6, 0)
        assert hidden.shape == normed.shape == (4, 8)
    args = _norm()
    args[1] = args[2] = args[3] = args[4] = None
    hidden, normed = nodes.gated_residual_norm(*args, 1.0, 1.0, 1e-6, 0)
    assert hidden.shape == (4, 8) and normed is None
    x = _ffn()
    x[0].requires_grad_(True)
    assert nodes.gated_ffn(*x, 0, 0).requires_grad
    with torch.no_grad():
        assert not nodes.gated_ffn(*x, 0, 0).requires_grad
