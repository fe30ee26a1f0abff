"""orthogonalize's arguments, without a GPU: what it refuses and what it hands
to the library, whose calls are replaced by a recorder."""
from __future__ import annotations

import struct
import types

import pytest


@pytest.fixture()
def calls(monkeypatch):
    """(in, out, ld_in, ld_out, rows, cols) of every matrix of every call."""
    import contextlib

    import torch
    from distributedspeed_amd import muon as M
    seen = []

    def run(table, count, *rest):
        seen.append([struct.unpack_from("=2Q4q", table, 48 * k) for k in range(count)])
        return 0

    lib = types.SimpleNamespace(dsx_orthogonalize_workspace=lambda table, n: 256, dsx_orthogonalize=run)
    monkeypatch.setattr(M.ops, "_device", lambda t: t.device)
    monkeypatch.setattr(M.ops, "stream_of", lambda dev: None)
    monkeypatch.setattr(M._lib, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    return seen


def test_inputs_whose_derivative_would_be_lost_are_refused(calls):
    import torch
    import torch.autograd.forward_ad as fw
    from distributedspeed_amd import orthogonalize
    g, p = torch.ones(4, 6), torch.nn.Parameter(torch.ones(4, 6))
    for args in ((p,), ([g, p],), (p * 2,), (torch.stack([p, p]),)):
        with pytest.raises(RuntimeError, match="not differentiable"):
            orthogonalize(*args)
    with pytest.raises(RuntimeError, match="not differentiable"):
        orthogonalize(g, out=torch.nn.Parameter(torch.ones(4, 6, dtype=torch.bfloat16)))
    with fw.dual_level():
        dual = fw.make_dual(g, g)
        for args in ((dual,), ([g, dual],)):
            with pytest.raises(RuntimeError, match="not differentiable"):
                orthogonalize(*args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="not differentiable"):
            orthogonalize(dual)
        orthogonalize(g)
    assert len(calls) == 1
    orthogonalize(p.detach())
    with torch.no_grad():
        assert not orthogonalize(p).requires_grad
        orthogonalize(g, out=torch.nn.Parameter(torch.ones(4, 6, dtype=torch.bfloat16)))
    assert len(calls) == 4


@pytest.mark.parametrize("shape,order", [((4, 2, 5, 7), (1, 0, 2, 3)), ((2, 3, 4, 5, 6), (2, 0, 1, 3, 4)),
                                         ((3, 5, 7), (0, 1, 2)), ((2, 2, 5, 7), (0, 1, 2, 3))])
def test_out_is_written_where_it_lies(calls, shape, order):
    """Batch dimensions in any order of memory: every matrix of `out` is a view of it."""
    import torch
    from distributedspeed_amd import orthogonalize
    out = torch.zeros(shape, dtype=torch.bfloat16).permute(order)
    updates = torch.ones(out.shape)
    assert orthogonalize(updates, out=out) is out
    rows, cols = out.shape[-2:]
    batch = [[]]
    for n in out.shape[:-2]:
        batch = [b + [k] for b in batch for k in range(n)]
    want = [(updates[tuple(b)].data_ptr(), out[tuple(b)].data_ptr(), cols, out.stride(-2), rows, cols) for b in batch]
    assert calls[-1] == want


def test_an_out_whose_matrices_share_memory_is_refused(calls):
    import torch
    from distributedspeed_amd import orthogonalize
    with pytest.raises(ValueError, match="overlap"):
        orthogonalize(torch.ones(3, 4, 5), out=torch.zeros(4, 5, dtype=torch.bfloat16).expand(3, 4, 5))
    with pytest.raises(ValueError, match="overlap"):
        orthogonalize(torch.ones(2, 3, 4, 5), out=torch.zeros(2, 1, 4, 5, dtype=torch.bfloat16).expand(2, 3, 4, 5))
    assert not calls


@pytest.mark.parametrize("shape", [(0, 4, 5), (2, 0, 4), (2, 4, 0), (2, 3, 0, 0), (0, 2, 3, 4), (2, 0, 3, 4), (0, 0, 4),
                                   (0, 0)])
def test_batches_of_empty_matrices_and_empty_batches(calls, shape):
    import torch
    from distributedspeed_amd import orthogonalize
    got = orthogonalize(torch.ones(shape))
    assert got.shape == shape and got.dtype == torch.bfloat16
    out = torch.zeros(shape, dtype=torch.bfloat16)
    assert orthogonalize(torch.ones(shape), out=out) is out


@pytest.mark.parametrize("n,m,count", [(14336, 4096, 1), (14336, 4096, 19), (14336, 4096, 200), (8192, 28672, 7),
                                       (64, 1 << 20, 40), (2048, 2048, 100), (3, 5, 4000)])
def test_scratch_is_bounded_for_any_length_of_list(n, m, count):
    """1 GiB, or what one matrix needs; beside it the records and the partial
    norms of every matrix (16 KiB at most) and the split sums (8 MiB)."""
    from distributedspeed_amd import _lib
    lib = _lib.load()
    for struct_, name in ((_lib.DsxMatrix, "dsx_orthogonalize_workspace"), (_lib.DsxMuonParam, "dsx_muon_workspace")):
        table = (struct_ * count)()
        for q in table:
            q.rows, q.cols = n, m
        s = (min(n, m) + 7) // 8 * 8
        one = 8 * (s * max(n, m) + 64) + 4 * (s * s + 256) + 8 * s + 1024
        got = getattr(lib, name)(table, count)
        assert 0 < got <= max(1 << 30, one) + count * (16384 + 32) + (8 << 20) + 1024
