"""What MuonOptimizer hands to the library, without a GPU: every pointer of the
table belongs to memory of the size the kernels walk, whatever state was
loaded and whatever became of the parameters since. The library's calls are
replaced by a recorder."""
from __future__ import annotations

import contextlib
import types

import pytest

F32, BF16, F16 = "float32", "bfloat16", "float16"


@pytest.fixture()
def muon(monkeypatch):
    """(MuonOptimizer, the recorded tables)."""
    import torch
    from distributedspeed_amd import muon as M
    tables = []

    def call(name, table, count, *rest):
        assert name == "dsx_muon_step" and count == len(table)
        tables.append(list(table))

    monkeypatch.setattr(M.ops, "_device", lambda t: t.device)
    monkeypatch.setattr(M.ops, "stream_of", lambda dev: None)
    monkeypatch.setattr(M._lib, "load", lambda: types.SimpleNamespace(dsx_muon_workspace=lambda table, n: 256))
    monkeypatch.setattr(M._lib, "call", call)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    return M.MuonOptimizer, tables


def _params(dtype, shapes=((6, 4), (3, 5)), value=0.5):
    import torch
    return [torch.nn.Parameter(torch.full(s, value, dtype=getattr(torch, dtype))) for s in shapes]


def _grads(params):
    for p in params:
        p.grad = p.detach().clone()


def _stepped(make, dtype, **kw):
    params = _params(dtype, **kw)
    opt = make(params, lr=0.01)
    _grads(params)
    opt.step()
    return params, opt


def _check_table(opt, params, table):
    """fp32 buffers of the parameter's own shape, contiguous; the parameter
    itself as the master where it is fp32 and as param16 where it is not."""
    import torch
    assert len(table) == len(params)
    for q, p in zip(table, params):
        st = opt.state[p]
        buffers = {"momentum_buffer"} | ({"master"} if p.dtype != torch.float32 else set())
        assert set(st) == buffers
        for key in buffers:
            t = st[key]
            assert t.dtype == torch.float32 and t.shape == p.shape and t.is_contiguous() and t.device == p.device
        assert q.momentum == st["momentum_buffer"].data_ptr()
        if p.dtype == torch.float32:
            assert q.master == p.data_ptr() and q.param16 is None
        else:
            assert q.master == st["master"].data_ptr() and q.param16 == p.data_ptr()
        assert (q.rows, q.cols) == tuple(p.shape)


@pytest.mark.parametrize("saved", [F32, BF16, F16])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_state_of_one_type_into_parameters_of_another(muon, saved, dtype):
    import torch
    make, tables = muon
    source, first = _stepped(make, saved, value=0.75)
    if saved != F32:
        for p in source:
            first.state[p]["master"].fill_(0.7512)
    for p in source:
        first.state[p]["momentum_buffer"].fill_(0.3001)
    params = _params(dtype)
    opt = make(params, lr=0.01)
    opt.load_state_dict(first.state_dict())
    _grads(params)
    opt.step()
    _check_table(opt, params, tables[-1])
    for p in params:
        assert bool((opt.state[p]["momentum_buffer"] == torch.tensor(0.3001)).all())
        # the weights go on from the master that was saved, or from the parameter where there was none
        weights = p.detach() if dtype == F32 else opt.state[p]["master"]
        assert bool((weights == torch.tensor(0.7512 if saved != F32 else 0.5)).all())


def test_state_of_torchs_muon(muon):
    import torch
    make, tables = muon
    source = _params(BF16)
    theirs = torch.optim.Muon(source, lr=0.125, weight_decay=0.25, adjust_lr_fn="match_rms_adamw")
    for p in source:
        theirs.state[p]["momentum_buffer"] = torch.full_like(p, 0.25)
    params = _params(BF16)
    opt = make(params, lr=0.01)
    opt.load_state_dict(theirs.state_dict())
    _grads(params)
    opt.step()
    _check_table(opt, params, tables[-1])
    group = opt.param_groups[0]
    assert group["lr"] == 0.125 and group["weight_decay"] == 0.25 and group["adjust_lr"] == "match_rms_adamw"
    assert all(bool((opt.state[p]["momentum_buffer"] == 0.25).all()) for p in params)


@pytest.mark.parametrize("before,after", [(F32, BF16), (BF16, F32), (BF16, F16)])
def test_parameters_cast_between_steps(muon, before, after):
    import torch
    make, tables = muon
    params, opt = _stepped(make, before)
    for p in params:
        p.grad = None
        p.data = p.data.to(getattr(torch, after))
    _grads(params)
    opt.step()
    _check_table(opt, params, tables[-1])
    opt.refresh_master()
    opt.step()
    _check_table(opt, params, tables[-1])


def test_refresh_master_of_a_parameter_that_became_fp32(muon):
    """Written from outside, the parameter wins over the master of its 16-bit past."""
    make, tables = muon
    params, opt = _stepped(make, BF16)
    for p in params:
        p.grad = None
        p.data = p.data.float().fill_(2.0)
    opt.refresh_master()
    _grads(params)
    opt.step()
    _check_table(opt, params, tables[-1])
    assert all(bool((p.detach() == 2.0).all()) for p in params)


@pytest.mark.parametrize("key", ["momentum_buffer", "master"])
def test_buffers_of_another_shape_are_refused_and_nothing_changes(muon, key):
    import copy

    import torch
    make, tables = muon
    params, opt = _stepped(make, BF16)
    state = copy.deepcopy(opt.state_dict())
    state["state"][1][key] = torch.zeros(2, 2)
    state["state"][0][key] += 1
    before = {p: {k: v.clone() for k, v in opt.state[p].items()} for p in params}
    with pytest.raises(ValueError, match=key):
        opt.load_state_dict(state)
    for p in params:
        assert all(torch.equal(opt.state[p][k], v) for k, v in before[p].items())
    count = len(tables)
    opt.state[params[0]][key] = torch.zeros(2, 2)
    with pytest.raises(ValueError, match=key):
        opt.step()
    opt.state[params[0]][key] = torch.zeros(6, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=key):
        opt.step()
    assert len(tables) == count


def test_saved_buffers_that_are_not_contiguous(muon):
    import copy

    import torch
    make, tables = muon
    params, opt = _stepped(make, BF16)
    state = copy.deepcopy(opt.state_dict())
    want = torch.arange(24.0).view(6, 4)
    for key in ("momentum_buffer", "master"):
        state["state"][0][key] = want.t().contiguous().t()
    opt.load_state_dict(state)
    opt.step()
    _check_table(opt, params, tables[-1])
    assert torch.equal(opt.state[params[0]]["momentum_buffer"], want) and torch.equal(opt.state[params[0]]["master"], want)


def test_saved_ids_that_are_not_counted_from_zero(muon):
    """The state belongs to a parameter by its group's list of ids."""
    import torch
    make, tables = muon
    params, opt = _stepped(make, BF16)
    for k, p in enumerate(params):
        opt.state[p]["momentum_buffer"].fill_(0.1001 * (k + 1))
    state = opt.state_dict()
    moved = {"state": {7: state["state"][0], 3: state["state"][1]},
             "param_groups": [{**state["param_groups"][0], "params": [7, 3]}]}
    others = _params(BF16)
    opt2 = make(others)
    opt2.load_state_dict(moved)
    _grads(others)
    opt2.step()
    _check_table(opt2, others, tables[-1])
    for k, p in enumerate(others):
        assert bool((opt2.state[p]["momentum_buffer"] == torch.tensor(0.1001 * (k + 1))).all())


def test_a_grad_of_another_shape_is_refused(muon):
    """A parameter that was replaced keeps the grad of its old shape."""
    import torch
    make, tables = muon
    params, opt = _stepped(make, F32)
    count = len(tables)
    params[0].data = torch.ones(60, 40)
    opt.state.pop(params[0])
    with pytest.raises(ValueError, match="grad"):
        opt.step()
    assert len(tables) == count


def test_a_grad_scale_elsewhere_is_refused(muon):
    """The kernels read it on the parameters' device."""
    import torch

    class Elsewhere(torch.Tensor):
        is_cuda = True
        device = torch.device("cuda", 1)

    make, tables = muon
    params, opt = _stepped(make, F32)
    count = len(tables)
    for scale in (torch.ones(1).as_subclass(Elsewhere), torch.ones(1, device="meta")):
        with pytest.raises(ValueError, match="grad_scale"):
            opt.step(grad_scale=scale)
    assert len(tables) == count
    opt.step(grad_scale=torch.ones(1))
    assert len(tables) == count + 1


def test_a_refused_group_is_not_added(muon):
    import torch
    make, tables = muon
    params, opt = _stepped(make, F32)
    good = torch.nn.Parameter(torch.ones(4, 4))
    for bad in (torch.nn.Parameter(torch.ones(5)), torch.nn.Parameter(torch.ones(4, 6).t()),
                torch.nn.Parameter(torch.ones(4, 4, dtype=torch.float64))):
        for group in ([bad], [good, bad], (p for p in (good, bad)), bad):
            with pytest.raises((ValueError, TypeError)):
                opt.add_param_group({"params": group})
            assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [good], "lr": 0.5})
    good.grad = torch.ones(4, 4)
    opt.step()
    assert len(opt.param_groups) == 2 and [len(t) for t in tables[-2:]] == [2, 1]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_buffer_saved_as_none_begins_anew(muon, dtype):
    import copy
    make, tables = muon
    params, opt = _stepped(make, dtype)
    state = copy.deepcopy(opt.state_dict())
    for s in state["state"].values():
        s.update(momentum_buffer=None, master=None)
    others = _params(dtype)
    opt2 = make(others)
    opt2.load_state_dict(state)
    _grads(others)
    opt2.step()
    _check_table(opt2, others, tables[-1])
    assert all(not bool(opt2.state[p]["momentum_buffer"].any()) for p in others)
