"""A batch's plan on another stream than the one it was made on."""
from __future__ import annotations

import copy

import pytest

pytestmark = pytest.mark.gpu


def _overlaps(tensors, ranges):
    return [t for t in tensors if any(t.data_ptr() < hi and lo < t.data_ptr() + t.nbytes for lo, hi in ranges)]


@pytest.mark.parametrize("copied", [False, True])
def test_a_plan_dropped_while_another_stream_reads_it(gpu, copied):
    """Made (or copied) on a stream that prepares batches, used on the current one behind queued
    work, and dropped: its memory is not handed out again on the first stream before
    that work has run, and the results are those of a plan that is kept."""
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention, rotary
    lengths = [300, 5, 0, 77]
    gen = torch.Generator("cuda").manual_seed(0)
    q, k, v = (torch.randn(382, h, 64, generator=gen, device="cuda").bfloat16().requires_grad_(True) for h in (4, 2, 2))
    dout = torch.randn(382, 4, 64, generator=gen, device="cuda").bfloat16()

    def run(packing):
        a, b = rotary(q, k, packing.positions)
        out = packed_attention(a, b, v, packing)
        return out, *torch.autograd.grad(out, (q, k, v), dout)

    kept = PackedSequences(lengths)
    kept.offsets
    want = run(kept)
    big = torch.randn(8192, 8192, device="cuda").bfloat16()
    prepare = torch.cuda.Stream()
    with torch.cuda.stream(prepare):
        packing = copy.deepcopy(kept) if copied else PackedSequences(lengths)
        made = [packing._tiles, packing.positions, packing.offsets]
        places = [(t.data_ptr(), t.data_ptr() + t.nbytes) for t in made]
        sizes = [t.nbytes for t in made]
    del made
    torch.cuda.synchronize()
    for _ in range(250):  # some 200 ms of products
        big @ big
    busy = torch.cuda.Event()
    got = run(packing)
    packing.offsets
    busy.record()
    del packing
    with torch.cuda.stream(prepare):
        later = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes * 8]
    assert not busy.query()  # the calls with the plan are still to run
    assert not _overlaps(later, places)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del later
    with torch.cuda.stream(prepare):  # and then it is free
        later = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes * 8]
    assert _overlaps(later, places)
