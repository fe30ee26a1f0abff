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

import struct

import torch

from . import _lib, ops

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}

# The argument blocks as bytes (DsxFfn and DsxNorm of include/dsx.h). These
# calls are a few microseconds of GPU time each for small inputs, so their host
# side is kept short: a block is packed once, the library's functions are bound
# once, and the autograd thread's part reuses what the forward worked out.
_FFN = struct.Struct("=4Q7q4i2Qq")
_NORM = struct.Struct("=5Q5qi3fQ")


class _Bound:
    """The library's functions, bound at first use."""

    def __getattr__(self, name: str):
        fn = getattr(_lib.load(), name)
        setattr(self, name, fn)
        return fn


_bound = _Bound()


def _raise(name: str, rc: int) -> None:
    raise _lib.DsxError(name, rc, _lib.last_error())


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [n, d], or a copy where its columns are not adjacent or its rows overlap."""
    if t.is_contiguous():
        return t
    (n, d), (row, col) = t.shape, t.stride()
    if (d > 1 and col != 1) or (n > 1 and row < d):
        return t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _scratch(nbytes: int, device: torch.device) -> torch.Tensor:
    if nbytes < 0:
        raise ValueError(_lib.last_error())
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _on(device: torch.device, run, *args):
    """run(*args) with `device` current."""
    if torch.cuda.current_device() == device.index:
        return run(*args)
    with torch.cuda.device(device):
        return run(*args)


def _refuse(name: str, t, first: torch.Tensor, optional: bool = False) -> None:
    """Why t cannot go with `first`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor" + (" or None" if optional else ""))
    if t.device != first.device:
        raise ValueError(f"{name} is on {t.device}, expected {first.device}")
    raise TypeError(f"{name} must be {first.dtype}, got {t.dtype}")


# ---- the gated feed-forward block ----------------------------------------------------------------

def _pack_ffn(x, w_gate, w_up, w_down, activation: int, keep: bool, saved: int, work: int, nbytes: int) -> bytes:
    f, d = w_gate.shape
    return _FFN.pack(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), _ld(x), _ld(w_gate),
                     _ld(w_up), _ld(w_down), x.shape[0], d, f, ops.dtype_code(x.dtype), activation, keep, 0, saved,
                     work, nbytes)


def _ffn_forward(x, w_gate, w_up, w_down, activation: int, keep: bool):
    """y, and the buffer the forward kept; x [tokens, width] and the weights row-contiguous."""
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    saved = _scratch(_bound.dsx_ffn_saved_bytes(x.shape[0], w_gate.shape[0], keep), dev)
    nbytes = _bound.dsx_ffn_workspace_bytes(_pack_ffn(x, w_gate, w_up, w_down, activation, keep, 0, 0, 0), 0)
    work = _scratch(nbytes, dev)
    q = _pack_ffn(x, w_gate, w_up, w_down, activation, keep, saved.data_ptr(), work.data_ptr(), nbytes)
    rc = _bound.dsx_ffn_forward(q, y.data_ptr(), y.shape[1], ops.stream_of(dev))
    if rc:
        _raise("dsx_ffn_forward", rc)
    return y, saved


def _ffn_backward(ctx, dy):
    x, w_gate, w_up, w_down, saved = ctx.saved_tensors
    dev, dy = x.device, _rows(dy)
    make = torch.empty if x.shape[0] else torch.zeros  # with no token the weights' gradients are zero
    grads = [make(t.shape, dtype=t.dtype, device=dev) if n else None
             for t, n in zip((x, w_gate, w_up, w_down), ctx.needs_input_grad)]
    nbytes = ctx.backward_bytes
    work = _scratch(nbytes, dev)
    q = _pack_ffn(x, w_gate, w_up, w_down, ctx.activation, True, saved.data_ptr(), work.data_ptr(), nbytes)
    at = [None if g is None else g.data_ptr() for g in grads]
    rc = _bound.dsx_ffn_backward(q, dy.data_ptr(), _ld(dy), at[0], x.shape[1], at[1], at[2], at[3], ops.stream_of(dev))
    if rc:
        _raise("dsx_ffn_backward", rc)
    return (*grads, None)


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        keep = any(ctx.needs_input_grad[:4])
        x, w_gate, w_up, w_down = _rows(x), _rows(w_gate), _rows(w_up), _rows(w_down)
        y, saved = _on(x.device, _ffn_forward, x, w_gate, w_up, w_down, activation, keep)
        if keep:
            ctx.save_for_backward(x, w_gate, w_up, w_down, saved)
            ctx.activation = activation
            ctx.backward_bytes = _bound.dsx_ffn_workspace_bytes(
                _pack_ffn(x, w_gate, w_up, w_down, activation, True, 0, 0, 0), 1)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            return _ffn_backward_once(ctx, dy)
        return _on(dy.device, _ffn_backward, ctx, dy)


@torch.autograd.function.once_differentiable
def _ffn_backward_once(ctx, dy):
    return _on(dy.device, _ffn_backward, ctx, dy)


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
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a tensor")
    dev = ops._device(x)
    ops.dtype_code(x.dtype)
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    for name, t in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if not isinstance(t, torch.Tensor) or t.dtype != x.dtype or t.device != dev:
            _refuse(name, t, x)
    d = x.shape[-1]
    if w_gate.dim() != 2:
        raise ValueError(f"w_gate must be [inner, width], got {tuple(w_gate.shape)}")
    f = w_gate.shape[0]
    if d < 1 or f < 1:
        raise ValueError(f"width and inner must be at least 1, got {d} and {f}")
    for name, t, shape in (("w_gate", w_gate, (f, d)), ("w_up", w_up, (f, d)), ("w_down", w_down, (d, f))):
        if t.shape != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    flat = x.reshape(-1, d) if x.dim() != 2 else x
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or w_down.requires_grad):
        y = _GatedFFN.apply(flat, w_gate, w_up, w_down, act)
    else:
        y, _ = _on(dev, _ffn_forward, _rows(flat), _rows(w_gate), _rows(w_up), _rows(w_down), act, False)
    return y.view(x.shape) if x.dim() != 2 else y


# ---- the norms around a block --------------------------------------------------------------------

def _at(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _norm_forward(residual, branch, post_weight, gate, next_weight, scales, keep: bool):
    """hidden, normed, the saved rstd and the packed arguments."""
    dev = residual.device
    rows, d = residual.shape
    hidden = torch.empty(residual.shape, dtype=residual.dtype, device=dev)
    normed = None if next_weight is None else torch.empty(residual.shape, dtype=residual.dtype, device=dev)
    rstd = torch.empty((2, rows), dtype=torch.float32, device=dev) if keep else None
    q = _NORM.pack(residual.data_ptr(), _at(branch), _at(post_weight), _at(gate), _at(next_weight), _ld(residual),
                   0 if branch is None else _ld(branch), rows, d, 0 if gate is None else gate.numel() // d,
                   ops.grad_code(residual.dtype), *scales, _at(rstd))
    rc = _bound.dsx_norm_forward(q, hidden.data_ptr(), None if normed is None else normed.data_ptr(),
                                 ops.stream_of(dev))
    if rc:
        _raise("dsx_norm_forward", rc)
    return hidden, normed, rstd, q


def _norm_backward(ctx, d_hidden, d_normed):
    saved = ctx.saved_tensors  # kept alive, and checked for changes in place; their addresses are in ctx.packed
    residual = saved[0]
    dev = residual.device
    make = torch.empty if residual.shape[0] else torch.zeros  # with no row the vectors' gradients are zero
    grads = [make(t.shape, dtype=t.dtype, device=dev) if t is not None and n else None
             for t, n in zip(saved, ctx.needs_input_grad[:5])]
    dh = dn = None
    ld_dh = ld_dn = 0
    if d_hidden is not None:
        d_hidden = _rows(d_hidden)
        dh, ld_dh = d_hidden.data_ptr(), _ld(d_hidden)
    if d_normed is not None:
        d_normed = _rows(d_normed)
        dn, ld_dn = d_normed.data_ptr(), _ld(d_normed)
    nbytes = ctx.backward_bytes
    work = _scratch(nbytes, dev)
    rc = _bound.dsx_norm_backward(ctx.packed, dh, ld_dh, dn, ld_dn,
                                  *[None if g is None else g.data_ptr() for g in grads], work.data_ptr(), nbytes,
                                  ops.stream_of(dev))
    if rc:
        _raise("dsx_norm_backward", rc)
    return (*grads, None)


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, post_weight, gate, next_weight, scales):
        keep = any(ctx.needs_input_grad[:5])
        residual = _rows(residual)
        if branch is not None:
            branch = _rows(branch)
        if post_weight is not None:
            post_weight = post_weight.contiguous()
        if gate is not None:
            gate = gate.contiguous()
        if next_weight is not None:
            next_weight = next_weight.contiguous()
        hidden, normed, rstd, q = _on(residual.device, _norm_forward, residual, branch, post_weight, gate, next_weight,
                                      scales, keep)
        ctx.set_materialize_grads(False)
        if keep:
            ctx.save_for_backward(residual, branch, post_weight, gate, next_weight, rstd)
            ctx.packed = q
            ctx.backward_bytes = _bound.dsx_norm_workspace_bytes(q)
        return hidden, normed

    @staticmethod
    def backward(ctx, d_hidden, d_normed):
        if d_hidden is None and d_normed is None:
            return (None,) * 6
        if torch.is_grad_enabled():
            return _norm_backward_once(ctx, d_hidden, d_normed)
        return _on((d_normed if d_hidden is None else d_hidden).device, _norm_backward, ctx, d_hidden, d_normed)


@torch.autograd.function.once_differentiable
def _norm_backward_once(ctx, d_hidden, d_normed):
    return _on((d_normed if d_hidden is None else d_hidden).device, _norm_backward, ctx, d_hidden, d_normed)


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
    if branch is None and (post_weight is not None or gate is not None):
        raise ValueError("post_weight and gate belong to a branch, and there is none")
    wants_grad = residual.requires_grad
    for name, t in (("branch", branch), ("post_weight", post_weight), ("gate", gate), ("next_weight", next_weight)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != residual.dtype or t.device != dev:
            _refuse(name, t, residual, True)
        wants_grad = wants_grad or t.requires_grad
    if branch is not None and branch.shape != residual.shape:
        raise ValueError(f"branch must be {list(residual.shape)}, got {list(branch.shape)}")
    for name, t in (("post_weight", post_weight), ("next_weight", next_weight)):
        if t is not None and t.shape != (d,):
            raise ValueError(f"{name} must be [{d}], got {list(t.shape)}")
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.shape[-1] != d or gate.numel() == 0:
            raise ValueError(f"gate must be [{d}] or [samples, {d}], got {list(gate.shape)}")
        rows = residual.numel() // d
        if gate.dim() == 2 and rows % gate.shape[0]:
            raise ValueError(f"gate has {gate.shape[0]} rows, which do not divide the {rows} rows")
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    scales = (float(branch_scale), float(residual_scale), float(eps))
    flat = residual if residual.dim() == 2 else residual.reshape(-1, d)
    flat_branch = branch if branch is None or branch.dim() == 2 else branch.reshape(-1, d)
    if wants_grad and torch.is_grad_enabled():
        hidden, normed = _GatedResidualNorm.apply(flat, flat_branch, post_weight, gate, next_weight, scales)
    else:
        vectors = [None if t is None else t.contiguous() for t in (post_weight, gate, next_weight)]
        hidden, normed, _, _ = _on(dev, _norm_forward, _rows(flat), None if branch is None else _rows(flat_branch),
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
