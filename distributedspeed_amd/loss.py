"""The loss of a language model as a differentiable GPU operator.

    linear_cross_entropy(x, weight, targets)   cross entropy of x weight^T

Both directions run the library's own kernels on the current stream, without a
host synchronisation, and never hold the logits. The forward can be captured into
a graph; a backward under capture is refused.
"""
from __future__ import annotations

import torch

from . import ops, sequence

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
MAX_DIM = 1 << 20
MAX_LOGITS = 1 << 38


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """The cross entropy of the logits x weight^T against `targets`, in fp32: x
    [..., width] and weight [vocab, width] (torch.nn.Linear's layout), both fp16
    or both bf16 on one GPU, targets [...] of int32 or int64. Rows whose target
    is `ignore_index` do not count: they take no part in the products, and their
    x may hold anything. `reduction` is "mean" (over the rows that count; NaN
    where there is none), "sum", or "none" (the rows' losses, zero in those that
    do not count). A row whose target is no row of `weight` has a loss of NaN,
    which reaches the gradients.

    The logits are fp32 sums that are reduced where they are computed. The
    backward computes them again, a piece of the vocabulary at a time, and
    rounds their gradients to the inputs' type for the two products. Rows of x
    and weight may be strided; a weight whose rows are not whole 16-byte chunks
    is copied first. At most 2^20 rows, width and vocab, and 2^38 logits.

    Differentiable once in x and weight, backwards (a forward-mode tangent is
    refused); results do not depend on timing. The backward keeps a copy of the
    rows of x that count."""
    code = REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a tensor")
    dev = ops._device(x)
    ops.dtype_code(x.dtype)
    if not isinstance(weight, torch.Tensor) or weight.dtype != x.dtype or weight.device != dev:
        sequence._refuse("weight", weight, x)
    if not isinstance(targets, torch.Tensor) or targets.dtype not in (torch.int32, torch.int64):
        raise TypeError("targets must be an int32 or int64 tensor")
    if targets.device != dev:
        raise ValueError(f"targets is on {targets.device}, expected {dev}")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"x must be [..., width] and weight [vocab, width], got {list(x.shape)} and "
                         f"{list(weight.shape)}")
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"targets must be {list(x.shape[:-1])}, got {list(targets.shape)}")
    d = x.shape[-1]
    if not (1 <= d <= MAX_DIM and 1 <= weight.shape[0] <= MAX_DIM and targets.numel() <= MAX_DIM):
        raise ValueError(f"width and vocab must lie in [1, {MAX_DIM}] and rows in [0, {MAX_DIM}]")
    if targets.numel() * weight.shape[0] > MAX_LOGITS:
        raise ValueError(f"rows * vocab must be at most 2^38, got {targets.numel()} * {weight.shape[0]}")
    ignore_index = int(ignore_index)
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError(f"ignore_index must fit 64 bits, got {ignore_index}")
    loss = (sequence._nodes or sequence._native()).linear_cross_entropy(
        x if x.dim() == 2 else x.reshape(-1, d), weight, targets.reshape(-1), ignore_index, code,
        ops.stream_of(dev).value or 0)
    return loss.view(targets.shape) if code == 0 else loss
