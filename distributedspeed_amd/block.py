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

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}

_nodes = None


def _native():
    """The autograd nodes (C++; see csrc/block_autograd.cpp), bound to the
    library's entry points at first use. There is no other path: where they
    are not built, this raises."""
    global _nodes
    if _nodes is None:
        lib = _lib.load()
        try:
            from . import _block_autograd as nodes
        except ImportError as e:
            raise RuntimeError("the block operators' autograd nodes are not built or do not load: run `python -c "
                               "'import __graft_entry__ as g; g.build()'` at the repository root") from e
        names = ("dsx_last_error", "dsx_ffn_saved_bytes", "dsx_ffn_workspace_bytes", "dsx_ffn_forward",
                 "dsx_ffn_backward", "dsx_norm_workspace_bytes", "dsx_norm_forward", "dsx_norm_backward")
        nodes.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names})
        _nodes = nodes
    return _nodes


def _refuse(name: str, t, first: torch.Tensor, optional: bool = False) -> None:
    """Why t cannot go with `first`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor" + (" or None" if optional else ""))
    if t.device != first.device:
        raise ValueError(f"{name} is on {t.device}, expected {first.device}")
    raise TypeError(f"{name} must be {first.dtype}, got {t.dtype}")


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """(act(x Wg^T) * (x Wu^T)) Wd^T for x [..., width], w_gate and w_up
    [inner, width] and w_down [width, inner] (torch.nn.Linear's layout), all
    fp16 or all bf16 on one GPU; `activation` is "silu", "gelu", "gelu_tanh" or
    "relu". Sums are fp32; the inner product act(g) u is rounded to the inputs'
    type once, or not at all for up to three tokens, so that a token's last
    bits depend on how many run with it. Rows may be strided; a tensor whose columns are not adjacent is
    copied first. Up to 2^20 tokens, none included.

    Differentiable once in all four tensors, backwards (a forward-mode tangent
    is refused). The backward keeps 8 bytes for every token and inner feature
    (10 for up to three tokens); without gradients nothing is kept."""
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
    y = (_nodes or _native()).gated_ffn(flat, w_gate, w_up, w_down, act, ops.stream_of(dev).value or 0)
    return y.view(x.shape) if x.dim() != 2 else y


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
    rows (at most 65533 samples). All tensors are of one type (fp32, fp16 or bf16) on one GPU. The
    arithmetic is fp32 and rounded once; normed is taken from hidden before its
    rounding. Rows may be strided.

    Differentiable once in all five tensors, backwards (a forward-mode tangent
    is refused); the backward computes hidden again
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
    for name, t in (("branch", branch), ("post_weight", post_weight), ("gate", gate), ("next_weight", next_weight)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != residual.dtype or t.device != dev:
            _refuse(name, t, residual, True)
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
    flat = residual if residual.dim() == 2 else residual.reshape(-1, d)
    flat_branch = branch if branch is None or branch.dim() == 2 else branch.reshape(-1, d)
    hidden, normed = (_nodes or _native()).gated_residual_norm(flat, flat_branch, post_weight, gate, next_weight,
                                                               branch_scale, residual_scale, eps,
                                                               ops.stream_of(dev).value or 0)
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
    steps, the others vectors. The forward takes fp16 or bf16 parameters and
    inputs: give a dtype, or leave the cast to the engine's fp16 or bf16 mode."""

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
