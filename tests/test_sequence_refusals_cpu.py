"""The attention, rotary and loss entry points without a GPU: sizes asked of the
library, the tile table, arguments that are refused before anything is launched,
and the wrappers' refusals of CPU tensors."""
from __future__ import annotations

import ctypes
import random

import pytest


@pytest.fixture(scope="module")
def lib():
    from distributedspeed_amd import _lib
    return _lib


def _tiles(L, lengths, capacity=None):
    table = (ctypes.c_int64 * max(1, len(lengths)))(*lengths)
    count = L.dsx_attention_tiles(table, len(lengths), None, 0)
    if count < 0:
        return None
    out = (ctypes.c_int32 * (8 * count + 1))()
    out[8 * count] = 77
    assert L.dsx_attention_tiles(table, len(lengths), out, count if capacity is None else capacity) == (
        count if capacity is None or capacity >= count else -1)
    assert out[8 * count] == 77
    rows = [tuple(out[4 * i:4 * i + 4]) for i in range(2 * count)]
    return rows[:count], rows[count:]


def test_tile_table(lib):
    """Every 128 rows of every sequence once in each half; the most work first: by
    queries those farthest from their sequence's first row, by keys from its end."""
    L = lib.load()
    rng = random.Random(0)
    lists = [[], [0], [1], [0, 0, 5], [128], [129, 128, 127], [5000]]
    lists += [[rng.choice((0, 1, 128, rng.randint(0, 3000))) for _ in range(rng.randint(1, 40))] for _ in range(60)]
    for lengths in lists:
        by_query, by_key = _tiles(L, lengths)
        want, first = [], 0
        for n in lengths:
            want += [(first + a, first, first + n, 0) for a in range(0, n, 128)]
            first += n
        assert sorted(by_query) == sorted(by_key) == sorted(want)
        far = [(r - s) // 128 for r, s, _, _ in by_query]
        assert far == sorted(far, reverse=True)
        far = [-(-(e - r) // 128) for r, _, e, _ in by_key]
        assert far == sorted(far, reverse=True)
    assert _tiles(L, [500, 3], capacity=3) is not None  # too small: refused, nothing written behind it
    for bad in ([-1], [5, -3], [2 ** 27, 1], [2 ** 62]):
        assert _tiles(L, bad) is None
        assert b"lengths" in L.dsx_last_error()
    assert L.dsx_attention_tiles(None, 2, None, 0) == -1 and L.dsx_attention_tiles(None, -1, None, 0) == -1


def _attention(lib, **kw):
    base = dict(q=4096, k=4096, v=4096, ld_q=256, ld_k=128, ld_v=128, head_q=64, head_k=64, head_v=64, tokens=300,
                tiles=4096, tile_count=4, heads=4, kv_heads=2, head_dim=64, dtype=2, causal=1, scale=0.125, longest=200)
    base.update(kw)
    return lib.DsxAttention(**base)


BAD_SIZES = [dict(dtype=0), dict(dtype=9), dict(tokens=-1), dict(tokens=2 ** 27 + 1), dict(heads=0), dict(kv_heads=0),
             dict(heads=5), dict(heads=1), dict(heads=2048, kv_heads=1), dict(head_dim=0), dict(head_dim=4),
             dict(head_dim=60), dict(head_dim=264), dict(tile_count=-1), dict(tile_count=0), dict(tile_count=301),
             dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(longest=-1),
             dict(longest=301), dict(tokens=2 ** 27, tile_count=2 ** 27), dict(tokens=2 ** 23, tile_count=2 ** 22),
             dict(pairs=-1), dict(pairs=60001)]
BAD_ROWS = [dict(q=None), dict(k=None), dict(v=None), dict(q=4104), dict(k=4098), dict(tiles=None), dict(tiles=4100),
            dict(ld_q=60), dict(ld_q=257), dict(ld_k=8), dict(ld_v=2 ** 24 + 8), dict(head_q=4), dict(head_k=63),
            dict(head_v=8)]


def test_attention_refusals(lib):
    L = lib.load()
    EINVAL = lib.DSX_EINVAL

    def forward(q, out=4096, lo=4096, lse=4096):
        return L.dsx_attention_forward(q, out, lo, lse, None)

    def backward(q, out=4096, lo=4096, lse=4096, do=4096, ld=256, head=64, grads=(4096,) * 3, ws=4096, nbytes=1 << 40):
        return L.dsx_attention_backward(q, out, lo, lse, do, ld, head, *grads, ws, nbytes, None)

    assert L.dsx_attention_workspace_bytes(ctypes.byref(_attention(lib))) >= 4 * 300 * 4
    for kw in BAD_SIZES:
        q = ctypes.byref(_attention(lib, **kw))
        assert L.dsx_attention_workspace_bytes(q) == -1, kw
        assert forward(q) == EINVAL and backward(q) == EINVAL, kw
    for kw in BAD_ROWS:
        q = ctypes.byref(_attention(lib, **kw))
        assert forward(q) == EINVAL and backward(q) == EINVAL, kw
    q = ctypes.byref(_attention(lib))
    assert forward(None) == EINVAL and backward(None) == EINVAL and L.dsx_attention_workspace_bytes(None) == -1
    for kw in (dict(out=None), dict(out=4100), dict(lo=4100), dict(lse=4098), dict(lo=None), dict(lse=None)):
        assert forward(q, **kw) == EINVAL and backward(q, **kw) == EINVAL, kw
    for kw in (dict(do=None), dict(do=4104), dict(ld=257), dict(ld=8), dict(head=8), dict(grads=(4104, 4096, 4096)),
               dict(grads=(4096, None, 4096)), dict(grads=(4096, 4096, None)), dict(grads=(4096, 4096, 4098)),
               dict(ws=None), dict(ws=4097), dict(nbytes=100)):
        assert backward(q, **kw) == EINVAL, kw
    empty = ctypes.byref(_attention(lib, tokens=0, tile_count=0, longest=0, q=None, k=None, v=None, tiles=None))
    assert forward(empty, None, None, None) == 0 and backward(empty, None, None, None, None, ws=None, nbytes=0) == 0


def test_attention_workspace_is_bounded(lib):
    """Parts take at most 512 MiB, whatever the tokens and heads."""
    L = lib.load()
    for tokens, heads, kv in ((300, 64, 1), (16384, 16, 2), (2 ** 20, 64, 8), (2 ** 24, 8, 8)):
        q = _attention(lib, tokens=tokens, heads=heads, kv_heads=kv, tile_count=-(-tokens // 128), longest=tokens, head_dim=128)
        assert 0 < L.dsx_attention_workspace_bytes(ctypes.byref(q)) <= 4 * tokens * heads + (512 << 20) + 8192


def _rotary(lib, **kw):
    base = dict(q=4096, k=4096, positions=4096, ld_q=256, ld_k=128, head_q=64, head_k=64, tokens=3, heads=4, kv_heads=2,
                head_dim=64, dims=64, dtype=2, interleaved=0, position_bytes=8, reserved=0, base=1e4)
    base.update(kw)
    return lib.DsxRotary(**base)


def test_rotary_refusals(lib):
    L = lib.load()
    for kw in (dict(dtype=7), dict(tokens=-1), dict(tokens=2 ** 27 + 1), dict(heads=0), dict(heads=1025),
               dict(kv_heads=-1), dict(kv_heads=1025), dict(head_dim=0), dict(head_dim=1025), dict(dims=66), dict(dims=-2),
               dict(dims=33), dict(base=0.0), dict(base=float("inf")), dict(base=float("nan")), dict(position_bytes=2),
               dict(q=None), dict(k=None), dict(positions=None), dict(q=4097), dict(k=4097), dict(positions=4100),
               dict(dtype=0, q=4098)):
        assert L.dsx_rotary(ctypes.byref(_rotary(lib, **kw)), 4096, 4096, 0, None) == lib.DSX_EINVAL, kw
    q = ctypes.byref(_rotary(lib))
    assert L.dsx_rotary(None, 4096, 4096, 0, None) == lib.DSX_EINVAL
    for out in ((None, 4096), (4096, None), (4097, 4096), (4096, 4097)):
        assert L.dsx_rotary(q, *out, 0, None) == lib.DSX_EINVAL
    assert L.dsx_rotary(ctypes.byref(_rotary(lib, tokens=0, q=None, k=None, positions=None)), None, None, 0, None) == 0


def _loss(lib, **kw):
    base = dict(x=4096, weight=4096, targets=4096, ld_x=64, ld_weight=64, tokens=50, width=64, vocab=1000, ignore_index=-100,
                dtype=2, target_bytes=8, reduction=1, reserved=0, saved=4096, workspace=4096, workspace_bytes=1 << 50)
    base.update(kw)
    return lib.DsxLoss(**base)


def test_loss_sizes_and_refusals(lib):
    L = lib.load()
    EINVAL = lib.DSX_EINVAL
    bad = [dict(dtype=0), dict(tokens=-1), dict(tokens=2 ** 20 + 1), dict(width=0), dict(width=2 ** 20 + 1), dict(vocab=0),
           dict(vocab=2 ** 20 + 1), dict(target_bytes=1), dict(reduction=3), dict(reduction=-1), dict(ld_weight=63)]
    for kw in bad:
        q = ctypes.byref(_loss(lib, **kw))
        assert L.dsx_loss_saved_bytes(q) == -1 and L.dsx_loss_workspace_bytes(q, 0) == -1, kw
        assert L.dsx_loss_forward(q, 4096, None) == EINVAL and L.dsx_loss_backward(q, 4096, 4096, 4096, None) == EINVAL, kw
    for kw in (dict(weight=None), dict(weight=4097), dict(saved=None), dict(saved=4100), dict(workspace=None),
               dict(workspace=4097), dict(workspace_bytes=64)):
        q = ctypes.byref(_loss(lib, **kw))
        assert L.dsx_loss_forward(q, 4096, None) == EINVAL and L.dsx_loss_backward(q, 4096, 4096, 4096, None) == EINVAL, kw
    for kw in (dict(x=None), dict(x=4097), dict(ld_x=63), dict(targets=None), dict(targets=4100),
               dict(target_bytes=4, targets=4098), dict(tokens=2 ** 20, vocab=2 ** 18 + 1)):
        assert L.dsx_loss_forward(ctypes.byref(_loss(lib, **kw)), 4096, None) == EINVAL, kw
    q = ctypes.byref(_loss(lib))
    assert L.dsx_loss_forward(None, 4096, None) == EINVAL and L.dsx_loss_saved_bytes(None) == -1
    assert L.dsx_loss_forward(q, None, None) == EINVAL and L.dsx_loss_forward(q, 4098, None) == EINVAL
    for args in ((None, 4096, 4096), (4098, 4096, 4096), (4096, 4097, 4096), (4096, 4096, 4097)):
        assert L.dsx_loss_backward(q, *args, None) == EINVAL


def test_loss_workspace_is_bounded(lib):
    """The logits' gradients take at most 512 MiB (or 1024 vocabulary rows'), an
    unaligned weight a copy more, and dx's sums 64 planes at most."""
    L = lib.load()
    for tokens, width, vocab in ((1, 64, 1000), (8192, 4096, 128256), (2 ** 20, 64, 2 ** 20), (100000, 1001, 50257)):
        q = _loss(lib, tokens=tokens, width=width, vocab=vocab, ld_x=width, ld_weight=width)
        nbytes = L.dsx_loss_workspace_bytes(ctypes.byref(q), 1)
        wide = -(-width // 8) * 8
        copy = vocab * wide * 2 if width % 8 else 0
        assert 0 < nbytes <= copy + max(512 << 20, 2048 * tokens) + 64 * tokens * wide * 4 + 4 * tokens + 4096
        assert L.dsx_loss_workspace_bytes(ctypes.byref(q), 0) > 0
        assert L.dsx_loss_saved_bytes(ctypes.byref(q)) >= tokens * (2 * wide + 20)


def test_wrappers_refuse_cpu_tensors():
    import torch
    from distributedspeed_amd import linear_cross_entropy, packed_attention, rotary
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises((ValueError, RuntimeError)):
        packed_attention(q, q, q, None)
    with pytest.raises((ValueError, RuntimeError)):
        rotary(q, q, torch.arange(4))
    with pytest.raises((ValueError, RuntimeError)):
        linear_cross_entropy(q[:, 0], q[:, 1], torch.zeros(4, dtype=torch.long))


def test_packed_sequences_refusals():
    from distributedspeed_amd import PackedSequences
    for bad in ([-1], [3, -2], [2 ** 27 + 1], [2 ** 27, 5]):
        with pytest.raises(ValueError):
            PackedSequences(bad, device="cuda:0")
    with pytest.raises(ValueError):
        PackedSequences([3], device="cpu")
    with pytest.raises((TypeError, ValueError)):
        PackedSequences(["a"], device="cuda:0")


def test_attention_block_refusals():
    from distributedspeed_amd import AttentionBlock
    for args in ((64, 3), (64, 0), (64, 4, 3), (64, 4, 0), (64, 4, 2, 15), (64, 4, 2, 258), (60, 4, 4)):
        with pytest.raises(ValueError):
            AttentionBlock(*args)
    block = AttentionBlock(64, 4, 2)
    assert block.head_dim == 16 and block.w_k.shape == (32, 64) and block.w_o.shape == (64, 64)
