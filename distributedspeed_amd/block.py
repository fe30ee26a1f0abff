"""A gated feed-forward block as differentiable GPU operators.

    gated_ffn(x, w_gate, w_up, w_down)            (act(x Wg^T) * (x Wu^T)) Wd^T
    gated_residual_norm(residual, branch, ...)    the norms before and after it,
                                                  with its gate and residual
    GatedFFNBlock                                 both as a module

Both directions run the library's own kernels on the current stream, without a
host synchronisation; the gradients work with torch.autograd and so with the
optimizers of this package.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, ops
from ._lib import DsxFfn, DsxNorm

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


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, post_weight, gate, next_weight, scales):
        keep = any(ctx.needs_input_grad[:5])
        residual = _rows(residual)
        branch = None if branch is None else _rows(branch)
        post_weight, gate, next_weight = (None if t is None else t.contiguous()
                                          for t in (post_weight, gate, next_weight))
        hidden, normed, rstd = _norm_forward(residual, branch, post_weight, gate, next_weight, scales, keep)
        ctx.set_materialize_grads(False)
        if keep:
            ctx.save_for_backward(residual, branch, post_weight, gate, next_weight, rstd)
            ctx.scales = scales
        return hidden, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_hidden, d_normed):
        *inputs, rstd = ctx.saved_tensors
        residual, dev = inputs[0], inputs[0].device
        if d_hidden is None and d_normed is None:
            return (None,) * 6
        d_hidden, d_normed = (None if t is None else _rows(t) for t in (d_hidden, d_normed))
        make = torch.empty if residual.shape[0] else torch.zeros  # with no row the vectors' gradients are zero
        grads = [make(t.shape, dtype=t.dtype, device=dev) if t is not None and need else None
                 for t, need in zip(inputs, ctx.needs_input_grad)]
        q = _describe_norm(*inputs, ctx.scales, rstd)
        with torch.cuda.device(dev):
            work = _scratch(_lib.load().dsx_norm_workspace_bytes(ctypes.byref(q)), dev)
            _lib.call("dsx_norm_backward", ctypes.byref(q), ops._ptr(d_hidden), 0 if d_hidden is None else _ld(d_hidden),
                      ops._ptr(d_normed), 0 if d_normed is None else _ld(d_normed), *(ops._ptr(g) for g in grads),
                      ops._ptr(work), work.numel(), ops.stream_of(dev))
        return (*grads, None)


def _describe_norm(residual, branch, post_weight, gate, next_weight, scales, rstd) -> DsxNorm:
    at = [None if t is None else t.data_ptr() for t in (residual, branch, post_weight, gate, next_weight)]
    rows, d = residual.shape
    gate_rows = 0 if gate is None else gate.numel() // d
    return DsxNorm(*at, _ld(residual), 0 if branch is None else _ld(branch), rows, d, gate_rows,
                   ops.grad_code(residual.dtype), *scales, None if rstd is None else rstd.data_ptr())


def _norm_forward(residual, branch, post_weight, gate, next_weight, scales, keep: bool):
    dev = residual.device
    hidden = torch.empty(residual.shape, dtype=residual.dtype, device=dev)
    normed = None if next_weight is None else torch.empty_like(hidden)
    rstd = torch.empty(2, residual.shape[0], dtype=torch.float32, device=dev) if keep else None
    q = _describe_norm(residual, branch, post_weight, gate, next_weight, scales, rstd)
    with torch.cuda.device(dev):
        _lib.call("dsx_norm_forward", ctypes.byref(q), ops._ptr(hidden), ops._ptr(normed), ops.stream_of(dev))
    return hidden, normed, rstd


def gated_residual_norm(residual: torch.Tensor, branch: torch.Tensor | None = None, *,
                        post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                        next_weight: torch.Tensor | None = None, branch_scale: float = 1.0,
                        residual_scale: float = 1.0, eps: float = 1e-6
                        ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(hidden, normed) around a block whose output is `branch`:

        z      = rms(branch) * post_weight        (branch, without post_weight)
        hidden = residual_scale * residual + branch_scale * gate * z
        normed = rms(hidden) * next_weight        (None, without next_weight)

    with rms(v) = v / sqrt(mean(v^2) + eps) over the last dimension. Without a
    branch it is the norm before a first block. residual and branch are
    [..., width], the weights [width]; gate is [width] (a value a channel) or
    [samples, width], whose i-th row serves the i-th of `samples` equal runs of
    rows. All tensors are of one type (fp32, fp16 or bf16) on one GPU. The
    arithmetic is fp32 and rounded once; normed is taken from hidden before its
    rounding. Rows may be strided.

    Differentiable once in all five tensors; the backward computes hidden again
    from the inputs and keeps 8 bytes a row beside them."""
    if not isinstance(residual, torch.Tensor):
        raise TypeError("residual must be a tensor")
    dev = ops._device(residual)
    ops.grad_code(residual.dtype)
    if residual.dim() < 1 or residual.shape[-1] < 1:
        raise ValueError(f"residual must be [..., width] with a width of at least 1, got {tuple(residual.shape)}")
    d = residual.shape[-1]
    rows = residual.numel() // d
    if branch is None and (post_weight is not None or gate is not None):
        raise ValueError("post_weight and gate belong to a branch, and there is none")
    for name, t in (("branch", branch), ("post_weight", post_weight), ("gate", gate), ("next_weight", next_weight)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or None")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev}")
        if t.dtype != residual.dtype:
            raise TypeError(f"{name} must be {residual.dtype}, got {t.dtype}")
    if branch is not None and branch.shape != residual.shape:
        raise ValueError(f"branch must be {list(residual.shape)}, got {list(branch.shape)}")
    for name, t in (("post_weight", post_weight), ("next_weight", next_weight)):
        if t is not None and tuple(t.shape) != (d,):
            raise ValueError(f"{name} must be [{d}], got {list(t.shape)}")
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.shape[-1] != d or gate.numel() == 0:
            raise ValueError(f"gate must be [{d}] or [samples, {d}], got {list(gate.shape)}")
        if gate.dim() == 2 and rows % gate.shape[0]:
            raise ValueError(f"gate has {gate.shape[0]} rows, which do not divide the {rows} rows")
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    scales = (float(branch_scale), float(residual_scale), float(eps))
    flat = residual if residual.dim() == 2 else residual.reshape(-1, d)
    flat_branch = branch if branch is None or branch.dim() == 2 else branch.reshape(-1, d)
    inputs = (flat, flat_branch, post_weight, gate, next_weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs):
        hidden, normed = _GatedResidualNorm.apply(*inputs, scales)
    else:
        vectors = (None if t is None else t.detach().contiguous() for t in inputs[2:])
        hidden, normed, _ = _norm_forward(_rows(flat.detach()), None if branch is None else _rows(flat_branch.detach()),
                                          *vectors, scales, False)
    if residual.dim() != 2:
        hidden = hidden.view(residual.shape)
        normed = None if normed is None else normed.view(residual.shape)
    return hidden, normed


class GatedFFNBlock(torch.nn.Module):
    """One block of a stack: (hidden, normed) -> (hidden, normed), where normed
    is the block's input and, in turn, the next block's:

        y      = gated_ffn(normed, w_gate, w_up, w_down)
        hidden = hidden + branch_scale * gate * rms(y) * post_weight
        normed = rms(hidden) * next_weight

    The stack begins with gated_residual_norm(x, next_weight=...). The gate is
    a value a channel; w_gate, w_up and w_down are the matrices that Muon
    steps, the others vectors."""

    def __init__(self, width: int, inner: int, *, activation: str = "silu", branch_scale: float = 1.0,
                 gate_init: float = 1.0, eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
        self.activation, self.branch_scale, self.eps = activation, float(branch_scale), float(eps)
        kw = dict(device=device, dtype=dtype)

        def matrix(rows, cols):
            return torch.nn.Parameter(torch.empty(rows, cols, **kw).normal_(std=cols ** -0.5))

        self.w_gate, self.w_up, self.w_down = matrix(inner, width), matrix(inner, width), matrix(width, inner)
        self.post_weight = torch.nn.Parameter(torch.ones(width, **kw))
        self.gate = torch.nn.Parameter(torch.full((width,), float(gate_init), **kw))
        self.next_weight = torch.nn.Parameter(torch.ones(width, **kw))

    def forward(self, hidden: torch.Tensor, normed: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        y = gated_ffn(normed, self.w_gate, self.w_up, self.w_down, activation=self.activation)
        return gated_residual_norm(hidden, y, post_weight=self.post_weight, gate=self.gate,
                                   next_weight=self.next_weight, branch_scale=self.branch_scale, eps=self.eps)
