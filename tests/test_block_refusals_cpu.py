"""The block and Muon entry points without a GPU: sizes asked of the library,
arguments it refuses before anything is launched, and the wrappers' refusals
of CPU tensors."""
from __future__ import annotations

import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from distributedspeed_amd import _lib
    return _lib


def _matrices(lib, shapes, ptr=4096, ld=None):
    table = (lib.DsxMatrix * len(shapes))()
    for q, (n, m) in zip(table, shapes):
        q.in_ = q.out = ptr
        q.ld_in = q.ld_out = m if ld is None else ld
        q.rows, q.cols = n, m
    return table


def test_orthogonalize_workspace_and_refusals(lib):
    L = lib.load()
    small, big = _matrices(lib, [(8, 8)]), _matrices(lib, [(8, 8)] * 100 + [(1000, 2000)])
    a, b = L.dsx_orthogonalize_workspace(small, 1), L.dsx_orthogonalize_workspace(big, 101)
    assert 0 < a < b and L.dsx_orthogonalize_workspace(None, 0) >= 0
    assert L.dsx_orthogonalize_workspace(_matrices(lib, [(-1, 3)]), 1) == -1
    assert L.dsx_orthogonalize_workspace(_matrices(lib, [(2 ** 20 + 1, 3)]), 1) == -1
    assert b"dimensions" in L.dsx_last_error()
    assert L.dsx_orthogonalize_workspace(None, 3) == -1
    coef = (ctypes.c_double * 15)(*([3.4445, -4.775, 2.0315] * 5))

    def call(table=small, n=1, dtype=2, steps=5, c=coef, eps=1e-7, ws=4096, nbytes=1 << 40):
        return L.dsx_orthogonalize(table, n, dtype, steps, c, eps, ws, nbytes, None)

    bad_coef = (ctypes.c_double * 15)(*([float("nan")] * 15))
    for kw in (dict(n=-1), dict(n=5000), dict(dtype=7), dict(steps=0), dict(steps=65), dict(c=None), dict(c=bad_coef),
               dict(eps=0.0), dict(eps=float("nan")), dict(ws=None), dict(ws=4097), dict(nbytes=16), dict(table=None),
               dict(table=_matrices(lib, [(8, 8)], ptr=None)), dict(table=_matrices(lib, [(8, 8)], ptr=4097)),
               dict(table=_matrices(lib, [(8, 8)], ld=7))):
        assert call(**kw) == lib.DSX_EINVAL, kw
    assert b"row stride" in L.dsx_last_error()


def test_muon_refusals(lib):
    L = lib.load()
    coef = (ctypes.c_double * 15)(*([3.4445, -4.775, 2.0315] * 5))

    def call(hyper=(0.95, 1.0, 1e-7, 1, 5), pdt=2, gdt=2, lr=0.1, mom=4096, grad=4096, ld=8, scale=None):
        table = (lib.DsxMuonParam * 1)(lib.DsxMuonParam(grad, mom, 4096, 4096, ld, 8, 8, lr, 0))
        return L.dsx_muon_step(table, 1, gdt, pdt, lib.DsxMuonHyper(*hyper), scale, coef, 4096, 1 << 40, None)

    for kw in (dict(hyper=(1.0, 1.0, 1e-7, 1, 5)), dict(hyper=(-0.1, 1.0, 1e-7, 1, 5)), dict(hyper=(0.9, 1.5, 1e-7, 1, 5)),
               dict(hyper=(0.9, 1.0, 0.0, 1, 5)), dict(hyper=(0.9, 1.0, 1e-7, 1, 0)), dict(pdt=0), dict(gdt=9),
               dict(lr=float("inf")), dict(mom=None), dict(mom=4100), dict(grad=4097), dict(ld=7), dict(scale=4097)):
        assert call(**kw) == lib.DSX_EINVAL, kw
    assert L.dsx_muon_workspace(None, 2) == -1


def _block(lib, **kw):
    base = dict(x=4096, w_gate=4096, w_up=4096, w_down=4096, ld_x=16, ld_gate=16, ld_up=16, ld_down=24, tokens=4,
                width=16, inner=24, dtype=2, activation=0, keep=1, reserved=0, saved=4096, workspace=4096,
                workspace_bytes=1 << 40)
    base.update(kw)
    return lib.DsxFfn(**base)


def test_ffn_sizes_and_refusals(lib):
    L = lib.load()
    assert L.dsx_ffn_saved_bytes(10, 24, 0) == 10 * 24 * 2 and L.dsx_ffn_saved_bytes(10, 23, 1) == 10 * 24 * 8
    assert L.dsx_ffn_saved_bytes(-1, 24, 0) == -1 and L.dsx_ffn_saved_bytes(1, 0, 0) == -1
    for tokens in (0, 1, 100, 5000):
        assert L.dsx_ffn_workspace_bytes(ctypes.byref(_block(lib, tokens=tokens)), 0) > 0
        assert L.dsx_ffn_workspace_bytes(ctypes.byref(_block(lib, tokens=tokens)), 1) >= 4 * tokens * 24
    assert L.dsx_ffn_workspace_bytes(None, 0) == -1
    bad = [dict(tokens=-1), dict(tokens=2 ** 20 + 1), dict(width=0), dict(inner=0), dict(dtype=0), dict(activation=4),
           dict(activation=-1), dict(x=None), dict(w_down=None), dict(w_up=4097), dict(saved=4100), dict(saved=None),
           dict(workspace=None), dict(ld_x=15), dict(ld_gate=15), dict(ld_up=1), dict(ld_down=23),
           dict(workspace_bytes=8)]
    for kw in bad:
        q = _block(lib, **kw)
        assert L.dsx_ffn_forward(ctypes.byref(q), 4096, 16, None) == lib.DSX_EINVAL, kw
        assert L.dsx_ffn_backward(ctypes.byref(q), 4096, 16, 4096, 16, None, None, None, None) == lib.DSX_EINVAL, kw
    q = _block(lib)
    assert L.dsx_ffn_forward(None, 4096, 16, None) == lib.DSX_EINVAL
    for y, ld in ((None, 16), (4097, 16), (4096, 15)):
        assert L.dsx_ffn_forward(ctypes.byref(q), y, ld, None) == lib.DSX_EINVAL
        assert L.dsx_ffn_backward(ctypes.byref(q), y, ld, None, 0, None, None, None, None) == lib.DSX_EINVAL
    assert L.dsx_ffn_backward(ctypes.byref(q), 4096, 16, 4097, 16, None, None, None, None) == lib.DSX_EINVAL
    assert L.dsx_ffn_backward(ctypes.byref(q), 4096, 16, None, 0, 4097, None, None, None) == lib.DSX_EINVAL
    assert L.dsx_ffn_backward(ctypes.byref(_block(lib, keep=0)), 4096, 16, None, 0, None, None, None, None) == lib.DSX_EINVAL
    empty = _block(lib, tokens=0, x=None, saved=None, workspace=None, workspace_bytes=0)
    assert L.dsx_ffn_forward(ctypes.byref(empty), None, 16, None) == 0


def _norm(lib, **kw):
    base = dict(residual=4096, branch=4096, post_weight=4096, gate=4096, next_weight=4096, ld_residual=16,
                ld_branch=16, rows=6, width=16, gate_rows=3, dtype=2, branch_scale=1.0, residual_scale=1.0, eps=1e-6,
                rstd=4096)
    base.update(kw)
    return lib.DsxNorm(**base)


def test_norm_sizes_and_refusals(lib):
    L = lib.load()
    assert L.dsx_norm_workspace_bytes(ctypes.byref(_norm(lib))) > 0
    assert L.dsx_norm_workspace_bytes(ctypes.byref(_norm(lib, rows=0))) > 0
    bad = [dict(dtype=5), dict(rows=-1), dict(rows=2 ** 28 + 1), dict(width=0), dict(width=2 ** 20 + 1),
           dict(branch=None), dict(gate_rows=0), dict(gate_rows=4), dict(gate_rows=65536, rows=65536),
           dict(eps=-1.0), dict(eps=float("nan"))]
    for kw in bad:
        assert L.dsx_norm_workspace_bytes(ctypes.byref(_norm(lib, **kw))) == -1, kw
        assert L.dsx_norm_forward(ctypes.byref(_norm(lib, **kw)), 4096, 4096, None) == lib.DSX_EINVAL, kw
    for kw in (dict(residual=None), dict(residual=4097), dict(gate=4097), dict(ld_residual=15), dict(ld_branch=15),
               dict(rstd=4098)):
        assert L.dsx_norm_forward(ctypes.byref(_norm(lib, **kw)), 4096, 4096, None) == lib.DSX_EINVAL, kw
    q = ctypes.byref(_norm(lib))
    assert L.dsx_norm_forward(None, 4096, 4096, None) == lib.DSX_EINVAL
    assert L.dsx_norm_forward(q, None, 4096, None) == lib.DSX_EINVAL
    assert L.dsx_norm_forward(q, 4096, None, None) == lib.DSX_EINVAL

    def back(args=q, dh=4096, ld_dh=16, dn=4096, ld_dn=16, grads=(4096,) * 5, ws=4096, nbytes=1 << 40):
        return L.dsx_norm_backward(args, dh, ld_dh, dn, ld_dn, *grads, ws, nbytes, None)

    assert back(ld_dh=15) == lib.DSX_EINVAL and back(ld_dn=3) == lib.DSX_EINVAL and back(dh=4097) == lib.DSX_EINVAL
    assert back(ws=None) == lib.DSX_EINVAL and back(ws=4097) == lib.DSX_EINVAL and back(nbytes=1) == lib.DSX_EINVAL
    assert back(grads=(4097,) + (4096,) * 4) == lib.DSX_EINVAL
    assert back(args=ctypes.byref(_norm(lib, rstd=None))) == lib.DSX_EINVAL
    assert back(args=ctypes.byref(_norm(lib, gate=None))) == lib.DSX_EINVAL  # a gradient of an input that is not there
    assert back(args=ctypes.byref(_norm(lib, rows=0)), dh=None, grads=(None,) * 5, ws=None, nbytes=0) == 0


def test_cpu_tensors_are_refused(lib):
    import torch
    from distributedspeed_amd import MuonOptimizer, gated_ffn, gated_residual_norm, orthogonalize
    x, w = torch.ones(4, 8, dtype=torch.bfloat16), torch.ones(8, 8, dtype=torch.bfloat16)
    for call in (lambda: gated_ffn(x, w, w, w), lambda: gated_residual_norm(x, x), lambda: orthogonalize(x),
                 lambda: MuonOptimizer([torch.nn.Parameter(x)])):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for bad in ((1.0, 2.0), ((1.0, 2.0, 3.0),) * 3, (float("nan"), 1.0, 1.0)):
        with pytest.raises(ValueError):
            orthogonalize(x, coefficients=bad)
    with pytest.raises(ValueError):
        gated_ffn(x, w, w, w, activation="swish")
