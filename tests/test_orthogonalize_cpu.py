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
