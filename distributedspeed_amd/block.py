"""A gated feed-forward block as differentiable GPU operators.

    gated_ffn(x, w_gate, w_up, w_down)            (act(x Wg^T) * (x Wu^T)) Wd^T

Both directions run the library's own kernels on the current stream, without a
host synchronisation; the gradients work with torch.autograd and so with the
optimizers of this package.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, ops
from ._lib import DsxFfn

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [n, d], or a copy where its columns are not adjacent or its rows overlap."""
    n, d = t.shape
    if (d > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < d):
        return t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _describe(x, w_gate, w_up, w_down, activation: int, keep: bool) -> DsxFfn:
    f, d = w_gate.shape
    return DsxFfn(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), _ld(x), _ld(w_gate), _ld(w_up),
                  _ld(w_down), x.shape[0], d, f, ops.dtype_code(x.dtype), activation, int(keep), 0, None, None, 0)


def _scratch(nbytes: int, device: torch.device) -> torch.Tensor:
    if nbytes < 0:
        raise ValueError(_lib.last_error())
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _forward(x, w_gate, w_up, w_down, activation: int, keep: bool):
    """y, and the buffer the forward kept; x [tokens, width] and the weights row-contiguous."""
    lib, dev = _lib.load(), x.device
    tokens, inner = x.shape[0], w_gate.shape[0]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    q = _describe(x, w_gate, w_up, w_down, activation, keep)
    with torch.cuda.device(dev):
        saved = _scratch(lib.dsx_ffn_saved_bytes(tokens, inner, int(keep)), dev)
        work = _scratch(lib.dsx_ffn_workspace_bytes(ctypes.byref(q), 0), dev)
        q.saved, q.workspace, q.workspace_bytes = saved.data_ptr(), work.data_ptr(), work.numel()
        _lib.call("dsx_ffn_forward", ctypes.byref(q), ops._ptr(y), y.shape[1], ops.stream_of(dev))
    return y, saved


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        keep = any(ctx.needs_input_grad[:4])
        x, w_gate, w_up, w_down = (_rows(t) for t in (x, w_gate, w_up, w_down))
        y, saved = _forward(x, w_gate, w_up, w_down, activation, keep)
        if keep:
            ctx.save_for_backward(x, w_gate, w_up, w_down, saved)
            ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w_gate, w_up, w_down, saved = ctx.saved_tensors
        need, dev = ctx.needs_input_grad, x.device
        dy = _rows(dy)
        make = torch.empty if x.shape[0] else torch.zeros  # with no token the weights' gradients are zero
        grads = [make(t.shape, dtype=t.dtype, device=dev) if n else None
                 for t, n in zip((x, w_gate, w_up, w_down), need)]
        q = _describe(x, w_gate, w_up, w_down, ctx.activation, True)
        with torch.cuda.device(dev):
            work = _scratch(_lib.load().dsx_ffn_workspace_bytes(ctypes.byref(q), 1), dev)
            q.saved, q.workspace, q.workspace_bytes = saved.data_ptr(), work.data_ptr(), work.numel()
            _lib.call("dsx_ffn_backward", ctypes.byref(q), ops._ptr(dy), _ld(dy), ops._ptr(grads[0]), x.shape[1],
                      *(ops._ptr(g) for g in grads[1:]), ops.stream_of(dev))
        return (*grads, None)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """(act(x Wg^T) * (x Wu^T)) Wd^T for x [..., width], w_gate and w_up
    [inner, width] and w_down [width, inner] (torch.nn.Linear's layout), all
    fp16 or all bf16 on one GPU; `activation` is "silu", "gelu", "gelu_tanh" or
    "relu". Sums are fp32; the inner product act(g) u is rounded to the inputs'
    type once. Rows may be strided; a tensor whose columns are not adjacent is
    copied first. Any number of tokens, none included.

    Differentiable once in all four tensors. The backward keeps 8 bytes for
    every token and inner feature; without gradients nothing is kept."""
    try:
        act = ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}") from None
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
    dev = ops._device(x)
    ops.dtype_code(x.dtype)
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    d = x.shape[-1]
    if w_gate.dim() != 2:
        raise ValueError(f"w_gate must be [inner, width], got {tuple(w_gate.shape)}")
    f = w_gate.shape[0]
    if d < 1 or f < 1:
        raise ValueError(f"width and inner must be at least 1, got {d} and {f}")
    for name, t, shape in (("w_gate", w_gate, (f, d)), ("w_up", w_up, (f, d)), ("w_down", w_down, (d, f))):
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev}")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} must be {x.dtype}, got {t.dtype}")
    flat = x.reshape(-1, d) if x.dim() != 2 else x
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down)):
        y = _GatedFFN.apply(flat, w_gate, w_up, w_down, act)
    else:
        y, _ = _forward(*(_rows(t.detach()) for t in (flat, w_gate, w_up, w_down)), act, False)
    return y.view(x.shape) if x.dim() != 2 else y
