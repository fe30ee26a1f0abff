"""Orthogonalisation of matrices by Newton-Schulz products, and the Muon
optimizer built on it.

    orthogonalize(updates)     the orthogonalised matrices, in bf16

For a matrix G with singular value decomposition U S V^T the iteration drives
every singular value of G / |G| towards 1 without computing the decomposition:
each step multiplies X by an odd polynomial a X + b (X X^T) X + c (X X^T)^2 X.
Muon's coefficients leave the singular values within about [0.7, 1.2] after
five steps, which is all the optimizer needs.
"""
from __future__ import annotations

import ctypes
import math
from typing import Sequence

import torch

from . import _lib, ops
from ._lib import DsxMatrix

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _coefficients(coefficients, steps: int) -> tuple[tuple[float, float, float], ...]:
    """One triple for every step, from one for all of them or one each."""
    rows = list(coefficients)
    if len(rows) == 3 and not any(isinstance(r, (tuple, list)) for r in rows):
        rows = [tuple(rows)] * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError(f"coefficients must be one triple, or {steps} of them (one for each step)")
    rows = tuple(tuple(float(v) for v in r) for r in rows)
    if not all(math.isfinite(v) for r in rows for v in r):
        raise ValueError("coefficients must be finite")
    return rows


def _check_ns(steps: int, eps: float) -> tuple[int, float]:
    steps, eps = int(steps), float(eps)
    if not 1 <= steps <= 64:
        raise ValueError(f"steps must be in [1, 64], got {steps}")
    if not 1e-20 <= eps <= 1.0:
        raise ValueError(f"eps must be in [1e-20, 1], got {eps}")
    return steps, eps


def _matrices(updates, name: str) -> list[torch.Tensor]:
    if isinstance(updates, torch.Tensor):
        if updates.dim() < 2:
            raise ValueError(f"{name} must have at least two dimensions, got {tuple(updates.shape)}")
        if updates.dim() == 2:
            return [updates]
        flat = updates.flatten(0, -3) if updates.numel() else updates.reshape(-1, *updates.shape[-2:])
        return list(flat.unbind(0))
    ms = list(updates)
    for t in ms:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or a sequence of tensors")
        if t.dim() != 2:
            raise ValueError(f"{name}: a list holds matrices, got a tensor of shape {tuple(t.shape)}")
    return ms


def _rows_contiguous(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy where its columns are not adjacent or its rows overlap."""
    if t.numel() and ((t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
        return t.contiguous()
    return t


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(1, t.shape[1])


def orthogonalize(updates: torch.Tensor | Sequence[torch.Tensor], *, steps: int = 5, coefficients=NS_COEFFICIENTS,
                  eps: float = 1e-7, out: torch.Tensor | Sequence[torch.Tensor] | None = None):
    """Newton-Schulz orthogonalisation of every matrix of `updates`: one
    tensor [..., rows, cols] or a sequence of matrices of any shapes, all
    fp32, fp16 or bf16 on one GPU. Returns bf16 of the same shape (a list for
    a sequence), or writes to `out`.

    `coefficients` is one (a, b, c) for all steps or one for each; they must
    keep the iterates' singular values below 4 (the iterates are fp16: their
    11 bits are why the result is bf16). A matrix whose norm is not finite
    becomes NaN; a zero matrix stays zero. A matrix whose columns are not
    adjacent is copied first. Runs on the current stream without a host
    synchronisation."""
    steps, eps = _check_ns(steps, eps)
    rows = _coefficients(coefficients, steps)
    ms = _matrices(updates, "updates")
    single = isinstance(updates, torch.Tensor)
    if not ms:
        if single:
            return updates.new_empty(updates.shape, dtype=torch.bfloat16) if out is None else out
        return []
    dev = ops._device(ms[0])
    code = ops.grad_code(ms[0].dtype)
    for t in ms:
        if t.device != dev:
            raise ValueError(f"updates are on {dev} and {t.device}")
        if t.dtype != ms[0].dtype:
            raise TypeError(f"updates are {ms[0].dtype} and {t.dtype}: pass one type at a time")
    if out is None:
        if single:
            result = torch.empty(updates.shape, dtype=torch.bfloat16, device=dev)
            outs = _matrices(result, "out")
        else:
            result = outs = [torch.empty(t.shape, dtype=torch.bfloat16, device=dev) for t in ms]
    else:
        result, outs = out, _matrices(out, "out")
        if len(outs) != len(ms):
            raise ValueError(f"out has {len(outs)} matrices, updates {len(ms)}")
        for t, o in zip(ms, outs):
            if o.shape != t.shape or o.dtype != torch.bfloat16 or o.device != dev:
                raise ValueError(f"out must be bfloat16 of shape {tuple(t.shape)} on {dev}, got {o.dtype} "
                                 f"{tuple(o.shape)} on {o.device}")
            if _rows_contiguous(o) is not o:
                raise ValueError("out must have adjacent columns and rows that do not overlap")
    ms = [_rows_contiguous(t.detach()) for t in ms]
    table = (DsxMatrix * len(ms))()
    for q, t, o in zip(table, ms, outs):
        q.in_, q.out, q.ld_in, q.ld_out = t.data_ptr(), o.data_ptr(), _row_stride(t), _row_stride(o)
        q.rows, q.cols = t.shape
    coef = (ctypes.c_double * (3 * steps))(*(v for r in rows for v in r))
    nbytes = _lib.load().dsx_orthogonalize_workspace(table, len(ms))
    if nbytes < 0:
        raise ValueError(_lib.last_error())
    with torch.cuda.device(dev):
        work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.call("dsx_orthogonalize", table, len(ms), code, steps, coef, eps, ops._ptr(work), nbytes,
                  ops.stream_of(dev))
    return result
