"""Orthogonalisation of matrices by Newton-Schulz products, and the Muon
optimizer built on it.

    orthogonalize(updates)     the orthogonalised matrices, in bf16
    MuonOptimizer(params)      the optimizer, for the matrices of a model

For a matrix G with singular value decomposition U S V^T the iteration drives
every singular value of G / |G| towards 1 without computing the decomposition:
each step multiplies X by an odd polynomial a X + b (X X^T) X + c (X X^T)^2 X.
Muon's coefficients leave the singular values within about [0.7, 1.2] after
five steps, which is all the optimizer needs.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Sequence

import torch
from torch.autograd import forward_ad

from . import _lib, ops
from ._lib import DsxMuonHyper, DsxMuonParam

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_MATRIX = struct.Struct("=2Q4q")  # DsxMatrix of include/dsx.h
_BUFFERS = ("momentum_buffer", "master")  # of a parameter's state: fp32, of its shape


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
        ms = [updates]
        for _ in range(updates.dim() - 2):  # views, whatever the batch dimensions' order in memory
            ms = [u for t in ms for u in t.unbind(0)]
        return ms
    ms = list(updates)
    for t in ms:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or a sequence of tensors")
        if t.dim() != 2:
            raise ValueError(f"{name}: a list holds matrices, got a tensor of shape {tuple(t.shape)}")
    return ms


def _refuse_tracked(ts: list[torch.Tensor]) -> None:
    """The kernels see values alone: a tensor that autograd follows, in either
    direction, would lose its derivative without a word."""
    tracked = torch.is_grad_enabled()
    for t in ts:
        if (tracked and t.requires_grad) or forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("orthogonalize is not differentiable: pass t.detach(), or call it under torch.no_grad()")


def _rows_contiguous(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy where its columns are not adjacent or its rows overlap."""
    if not t.is_contiguous() and t.numel() and ((t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
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
    11 bits are why the result is bf16). A matrix with an element that is not
    finite becomes NaN; a zero matrix stays zero. At most 4096 matrices a call,
    with sides of at most 2^20. Each step also multiplies, by its `a`, what the
    iterates' roundings put where the matrix has nothing: an fp32 matrix of rank
    four is 4e-3 off after five steps of Muon's coefficients, 1e-2 after six and
    1e-1 after eight (128 x 128; singular values over 10^4: 2e-3, 3e-3, 5e-3).
    Matrices with a side of at most 64 stay in fp32 (7e-4 beside the result's
    own rounding after eight). A norm far below eps (1e-5 of it) leaves the fp16
    iterates little of their bits. A matrix whose columns are not
    adjacent is copied first. Not differentiable: a tensor that requires grad
    (while grad mode is on) or carries a forward-mode tangent is refused. Runs
    on the current stream without a host synchronisation."""
    steps, eps = _check_ns(steps, eps)
    rows = _coefficients(coefficients, steps)
    ms = _matrices(updates, "updates")
    single = isinstance(updates, torch.Tensor)
    if not ms:
        if single:
            return updates.new_empty(updates.shape, dtype=torch.bfloat16) if out is None else out
        return []
    _refuse_tracked(ms)
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
        _refuse_tracked(outs)
        if isinstance(out, torch.Tensor) and any(n > 1 and k == 0 for n, k in zip(out.shape, out.stride())):
            raise ValueError("out's matrices must not overlap")
        if len(outs) != len(ms):
            raise ValueError(f"out has {len(outs)} matrices, updates {len(ms)}")
        for t, o in zip(ms, outs):
            if o.shape != t.shape or o.dtype != torch.bfloat16 or o.device != dev:
                raise ValueError(f"out must be bfloat16 of shape {tuple(t.shape)} on {dev}, got {o.dtype} "
                                 f"{tuple(o.shape)} on {o.device}")
            if _rows_contiguous(o) is not o:
                raise ValueError("out must have adjacent columns and rows that do not overlap")
    ms = [_rows_contiguous(t) for t in ms]
    table = b"".join(_MATRIX.pack(t.data_ptr(), o.data_ptr(), _row_stride(t), _row_stride(o), *t.shape)
                     for t, o in zip(ms, outs))
    coef = struct.pack(f"={3 * steps}d", *(v for r in rows for v in r))
    lib = _lib.load()
    nbytes = lib.dsx_orthogonalize_workspace(table, len(ms))
    if nbytes < 0:
        raise ValueError(_lib.last_error())

    def run():
        work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = lib.dsx_orthogonalize(table, len(ms), code, steps, coef, eps, work.data_ptr(), nbytes, ops.stream_of(dev))
        if rc:
            raise _lib.DsxError("dsx_orthogonalize", rc, _lib.last_error())

    if torch.cuda.current_device() == dev.index:
        run()
    else:
        with torch.cuda.device(dev):
            run()
    return result


class MuonOptimizer(torch.optim.Optimizer):
    """Muon for matrix parameters, with torch.optim.Muon's arguments (but
    adjust_lr, which is adjust_lr_fn there) and its state dicts:

        buf = momentum * buf + (1 - momentum) * grad
        u   = momentum * buf + (1 - momentum) * grad   (nesterov; else buf)
        w   = w * (1 - lr * weight_decay) - lr * factor * orthogonalize(u)

    where factor is sqrt(max(1, rows / cols)) for adjust_lr "original" and
    0.2 * sqrt(max(rows, cols)) for "match_rms_adamw", which lets AdamW's
    learning rate and weight decay carry over. Parameters are 2-D and
    contiguous; fp16 and bf16 ones get an fp32 master (state[p]["master"])
    that the step updates and rounds to the parameter, in the launch that
    forms the last Newton-Schulz product: the orthogonalised update is never
    written to memory. Vectors, embeddings and output heads belong to another
    optimizer (AdamWOptimizer).

    step(grad_scale=...) divides the grads by a one-element fp32 tensor on
    their device (AdamWOptimizer.loss_scale_tensor(), before that optimizer's
    own step, which may move it). A grad that is not finite skips the step of
    its param group (and type): nothing of it changes, and last_step_skipped()
    says so. It moves no loss scale: an AdamWOptimizer beside it sees its own
    grads alone, so under a dynamic scale the caller has to halve it where only
    a matrix's grad overflowed:

        muon.step(grad_scale=adamw.loss_scale_tensor())
        if muon.last_step_skipped():  # synchronises
            adamw.set_scaler_state(adamw.read_state().scale / 2)
        else:
            adamw.step()

    step() does not synchronise the host with the device."""

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95,
                 nesterov: bool = True, ns_coefficients=NS_COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5,
                 adjust_lr: str = "original"):
        if not 0.0 <= lr or not math.isfinite(lr):
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"Invalid momentum value: {momentum}")
        if adjust_lr not in ("original", "match_rms_adamw"):
            raise ValueError(f"adjust_lr must be 'original' or 'match_rms_adamw', got {adjust_lr!r}")
        ns_steps, eps = _check_ns(ns_steps, eps)
        _coefficients(ns_coefficients, ns_steps)
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=bool(nesterov),
                                      ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps,
                                      adjust_lr=adjust_lr))
        self._skips: list[torch.Tensor] = []

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            for p in self.param_groups[-1]["params"]:
                ops._device(p)
                ops.grad_code(p.dtype)
                if p.dim() != 2:
                    raise ValueError(f"Muon steps matrices; got a parameter of shape {tuple(p.shape)}")
                if not p.is_contiguous():
                    raise ValueError("Muon's parameters must be contiguous")
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    def __setstate__(self, state: dict) -> None:
        """Groups as this class has them, also from torch.optim.Muon's state
        dict, whose adjust_lr_fn is adjust_lr here (None: "original")."""
        super().__setstate__(state)
        self._skips = []
        for g in self.param_groups:
            if "adjust_lr" not in g:
                g["adjust_lr"] = g.pop("adjust_lr_fn", None) or "original"

    def _state_of(self, p: torch.Tensor) -> dict:
        """p's buffers as the step needs them for p's type of now: a momentum,
        and a master where p is 16-bit. The state may have been loaded from a
        run of another type, or p cast since the last step: a 16-bit p without
        a master begins one from its own values, an fp32 p takes the values of
        a master left over and goes on without it. The kernels walk every
        buffer by p's shape, so anything else is refused."""
        st = self.state[p]
        for key in _BUFFERS:
            if key in st and st[key] is None:
                del st[key]
        if "momentum_buffer" not in st:
            st["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if p.dtype != torch.float32 and "master" not in st:
            st["master"] = p.detach().float()
        for key in _BUFFERS:
            t = st.get(key)
            if t is not None and (t.shape != p.shape or t.dtype != torch.float32 or t.device != p.device
                                  or not t.is_contiguous()):
                raise ValueError(f"{key} must be a contiguous fp32 tensor of shape {tuple(p.shape)} on {p.device}, got "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
        if p.dtype == torch.float32 and "master" in st:
            p.copy_(st.pop("master"))
        return st

    @torch.no_grad()
    def refresh_master(self) -> None:
        """Take the fp32 masters from the current params (after they were
        written from outside the step, as by a module's load_state_dict)."""
        for p, st in self.state.items():
            if p.dtype == torch.float32:
                st.pop("master", None)
            elif "master" in st:
                st["master"].copy_(p)

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: torch.Tensor | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if grad_scale is not None and (not isinstance(grad_scale, torch.Tensor) or grad_scale.numel() != 1
                                       or grad_scale.dtype != torch.float32):
            raise ValueError("grad_scale must be a one-element float32 tensor")
        self._skips = []
        for g in self.param_groups:
            lists: dict[tuple, list[torch.Tensor]] = {}
            for p in g["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not support sparse gradients")
                if p.grad.shape != p.shape or p.grad.device != p.device:
                    raise ValueError(f"a grad of shape {tuple(p.grad.shape)} on {p.grad.device} for a parameter of "
                                     f"shape {tuple(p.shape)} on {p.device}")
                lists.setdefault((p.device, p.grad.dtype, p.dtype), []).append(p)
            for (dev, gdt, pdt), ps in lists.items():
                self._step_list(g, dev, gdt, pdt, ps, grad_scale)
        return loss

    def _step_list(self, g: dict, dev, gdt, pdt, ps: list, grad_scale) -> None:
        if grad_scale is not None and grad_scale.device != dev:
            raise ValueError(f"grad_scale is on {grad_scale.device}, the parameters on {dev}")
        lr, steps = float(g["lr"]), int(g["ns_steps"])
        decay = 1.0 - lr * g["weight_decay"]
        if not 0.0 <= decay <= 1.0:
            raise ValueError(f"lr * weight_decay must be in [0, 1], got {lr * g['weight_decay']}")
        table = (DsxMuonParam * len(ps))()
        grads = [_rows_contiguous(p.grad) for p in ps]
        for q, p, gr in zip(table, ps, grads):
            if not p.is_contiguous():
                raise ValueError("Muon's parameters must be contiguous")
            st = self._state_of(p)
            rows, cols = p.shape
            factor = (0.2 * math.sqrt(max(rows, cols)) if g["adjust_lr"] == "match_rms_adamw"
                      else math.sqrt(max(1.0, rows / cols)) if cols else 1.0)
            q.grad, q.momentum = gr.data_ptr(), st["momentum_buffer"].data_ptr()
            if pdt == torch.float32:
                q.master = p.data_ptr()
            else:
                q.master, q.param16 = st["master"].data_ptr(), p.data_ptr()
            q.ld_grad, q.rows, q.cols, q.lr = _row_stride(gr), rows, cols, lr * factor
        coef = (ctypes.c_double * (3 * steps))(*(v for r in _coefficients(g["ns_coefficients"], steps) for v in r))
        hyper = DsxMuonHyper(float(g["momentum"]), decay, float(g["eps"]), int(g["nesterov"]), steps)
        nbytes = _lib.load().dsx_muon_workspace(table, len(ps))
        if nbytes < 0:
            raise ValueError(_lib.last_error())
        with torch.cuda.device(dev):
            work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            skip = work[:4].view(torch.int32)
            _lib.call("dsx_muon_step", table, len(ps), ops.grad_code(gdt),
                      ops.dtype_code(torch.float16 if pdt == torch.float32 else pdt), hyper, ops._ptr(grad_scale), coef,
                      ops._ptr(work), nbytes, ops.stream_of(dev))
            self._skips.append(skip.clone())

    def last_step_skipped(self) -> bool:
        """Whether any part of the last step was skipped (synchronises)."""
        return any(bool(s.item()) for s in self._skips)

    def load_state_dict(self, state_dict: dict) -> None:
        """torch's, but the fp32 state stays fp32 for 16-bit parameters. A
        buffer of another shape than its parameter's is refused (ValueError)
        before anything changes. State of a run of another parameter type is
        taken over by the next step (see _state_of)."""
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        pairs = [(p, state_dict["state"].get(i, {})) for i, p in
                 zip(ids, (p for g in self.param_groups for p in g["params"]))]
        for p, saved in pairs:
            for key in _BUFFERS:
                t = saved.get(key)
                if t is not None and tuple(t.shape) != tuple(p.shape):
                    raise ValueError(f"{key} has shape {tuple(t.shape)}, its parameter {tuple(p.shape)}")
        super().load_state_dict(state_dict)
        for p, saved in pairs:
            for key in _BUFFERS:
                if saved.get(key) is not None:
                    self.state[p][key] = saved[key].detach().to(device=p.device, dtype=torch.float32, copy=True,
                                                                memory_format=torch.contiguous_format)
