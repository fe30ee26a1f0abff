"""Attention over packed sequences as differentiable GPU operators.

    PackedSequences(lengths)               where the sequences of a batch lie
    rotary(q, k, positions)                queries and keys turned by position
    packed_attention(q, k, v, packing)     softmax(scale q k^T) v within each
    AttentionBlock                         these between projections, as a module

Both directions run the library's own kernels on the current stream, without a
host synchronisation; the gradients work with torch.autograd and so with the
optimizers of this package. Forwards can be captured into a graph; a backward
under capture is refused.
"""
from __future__ import annotations

import ctypes
import math
import operator

import numpy as np
import torch

from . import _lib, ops
from .block import gated_residual_norm

MAX_TOKENS, MAX_HEADS, MAX_HEAD_DIM, MAX_ROTARY_DIM = 1 << 27, 1024, 256, 1024
MAX_TILES = 1 << 24  # of 128 rows, times heads

_nodes = None


def _native():
    """The autograd nodes (C++; see csrc/sequence_autograd.cpp), bound to the
    library's entry points at first use. There is no other path: where they
    are not built, this raises."""
    global _nodes
    if _nodes is None:
        lib = _lib.load()
        try:
            from . import _sequence_autograd as nodes
        except ImportError as e:
            raise RuntimeError("the sequence operators' autograd nodes are not built or do not load: run `python -c "
                               "'import __graft_entry__ as g; g.build()'` at the repository root") from e
        names = ("dsx_last_error", "dsx_stream_capturing", "dsx_attention_forward", "dsx_attention_workspace_bytes",
                 "dsx_attention_backward", "dsx_rotary", "dsx_loss_saved_bytes", "dsx_loss_workspace_bytes", "dsx_loss_forward",
                 "dsx_loss_backward")
        nodes.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names})
        _nodes = nodes
    return _nodes


class PackedSequences:
    """Where the sequences of a batch lie: of the given lengths (host integers,
    zero allowed), one behind the other from row 0. Made once for a batch and
    used by all its layers, in both directions, on any stream of `device`; it may
    be dropped as soon as the calls with it are made. It holds the kernels' tile
    table, so that a captured graph needs it alive. positions and offsets are made
    at their first use, which belongs before a capture.

        lengths   as a tuple
        tokens    their sum
        positions int32 [tokens]: each row's place in its sequence
        offsets   int32 [sequences + 1]: first rows, and the end"""

    def __init__(self, lengths, *, device=None):
        lengths = [operator.index(n) for n in (lengths.tolist() if isinstance(lengths, (torch.Tensor, np.ndarray)) else lengths)]
        if any(n < 0 for n in lengths) or sum(lengths) > MAX_TOKENS:
            raise ValueError(f"lengths must be at least 0 and add up to at most {MAX_TOKENS}")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError(f"device must be a GPU, got {device}")
        self.lengths = tuple(lengths)
        self.tokens = sum(lengths)
        self._longest, self._pairs = max(lengths, default=0), sum(n * n for n in lengths)
        self.device = torch.device("cuda", torch.cuda.current_device()) if device.index is None else device
        self._seen = set()  # (address, stream) of its tensors and the streams that the allocator knows of
        self._tiles = self._made(_tile_table(lengths))
        self._positions = self._offsets = None

    def __repr__(self) -> str:
        return f"PackedSequences({len(self.lengths)} sequences, {self.tokens} tokens, {self.device})"

    def _made(self, values: np.ndarray) -> torch.Tensor:
        """On the device when this returns, for any stream of it."""
        t = torch.from_numpy(values).to(self.device)
        self._seen.add((t.data_ptr(), ops.stream_of(self.device).value or 0))
        return t

    def _on_stream(self, t: torch.Tensor, stream: int) -> torch.Tensor:
        """t for work on `stream`, the current one: where it was made on another, its
        memory is not handed out again before what is queued by the time it is
        dropped has run. (A graph's replays come later: it needs t alive.)"""
        use = (t.data_ptr(), stream)
        if use not in self._seen:
            t.record_stream(torch.cuda.current_stream(self.device))
            self._seen.add(use)
        return t

    @property
    def positions(self) -> torch.Tensor:
        if self._positions is None:
            first = np.cumsum([0, *self.lengths], dtype=np.int64)[:-1]
            at = np.arange(self.tokens, dtype=np.int64) - np.repeat(first, self.lengths)
            self._positions = self._made(at.astype(np.int32))
        return self._on_stream(self._positions, ops.stream_of(self.device).value or 0)

    @property
    def offsets(self) -> torch.Tensor:
        if self._offsets is None:
            self._offsets = self._made(np.cumsum([0, *self.lengths]).astype(np.int32))
        return self._on_stream(self._offsets, ops.stream_of(self.device).value or 0)


def _tile_table(lengths) -> np.ndarray:
    """The kernels' tile table of sequences of these lengths, int32 [2, count, 4]."""
    lib = _lib.load()
    table = (ctypes.c_int64 * len(lengths))(*lengths)
    count = lib.dsx_attention_tiles(table, len(lengths), None, 0)
    if count < 0:
        raise ValueError(_lib.last_error())
    tiles = np.empty((2, count, 4), np.int32)
    if lib.dsx_attention_tiles(table, len(lengths), tiles.ctypes.data, count) != count:
        raise ValueError(_lib.last_error())
    return tiles


def _refuse(name: str, t, first: torch.Tensor) -> None:
    """Why t cannot go with `first`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device != first.device:
        raise ValueError(f"{name} is on {t.device}, expected {first.device}")
    raise TypeError(f"{name} must be {first.dtype}, got {t.dtype}")


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, packing: PackedSequences, *,
                     causal: bool = True, scale: float | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v within each sequence of `packing`, over the keys up
    to the query's own where `causal`: q [rows, heads, head_dim], k and v [rows,
    kv_heads, head_dim], all fp16 or all bf16 on one GPU; heads is a multiple of
    kv_heads, and query head h reads key head h // (heads // kv_heads). head_dim
    is at most 256, scale 1 / sqrt(head_dim) unless given (2^-126 to 1e38), and the
    sequences' tiles of 128 rows times heads below 2^24. rows may be more than
    packing.tokens: the rest hold anything, and zeros in the result and in the
    gradients.

    Scores, statistics and sums are fp32; the probabilities are rounded to the
    inputs' type for the product with v. (Scaled scores of 2^24 and more, which fp32
    does not tell apart by one, may give NaN.) Rows and heads may be strided (the
    parts of one projection's rows); tensors whose features are not adjacent,
    not a multiple of eight or not 16-byte aligned are copied first. Sequences
    do not see each other: a value that is not finite stays within its own,
    where it may reach any row.

    Differentiable once in q, k and v, backwards (a forward-mode tangent is
    refused); results do not depend on timing, but in their last bits on how much
    other work a batch holds, by which it is shared out. The backward keeps the output
    twice (its rounding errors too) and 4 bytes a row and head beside the
    inputs."""
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a tensor")
    dev = ops._device(q)
    ops.dtype_code(q.dtype)
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dtype != q.dtype or t.device != dev:
            _refuse(name, t, q)
    if not isinstance(packing, PackedSequences):
        raise TypeError("packing must be PackedSequences")
    if packing.device != dev:
        raise ValueError(f"packing is on {packing.device}, expected {dev}")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k must be [rows, heads, head_dim], got {list(q.shape)} and {list(k.shape)}")
    rows, heads, d = q.shape
    kv_heads = k.shape[1]
    if k.shape != (rows, kv_heads, d) or v.shape != k.shape:
        raise ValueError(f"k and v must be [{rows}, kv_heads, {d}], got {list(k.shape)} and {list(v.shape)}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads or heads > MAX_HEADS:
        raise ValueError(f"heads must be a multiple of kv_heads and at most {MAX_HEADS}, got {heads} and {kv_heads}")
    if not 1 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must lie in [1, {MAX_HEAD_DIM}], got {d}")
    if rows < packing.tokens:
        raise ValueError(f"q has {rows} rows, packing {packing.tokens} tokens")
    scale = 1 / math.sqrt(d) if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= 1e38:
        raise ValueError(f"scale must lie in [2^-126, 1e38], got {scale}")
    if packing._tiles.shape[1] * heads >= MAX_TILES:
        raise ValueError(f"tiles times heads must be below 2^24, got {packing._tiles.shape[1]} * {heads}")
    stream = ops.stream_of(dev).value or 0
    tiles = packing._on_stream(packing._tiles, stream)
    return (_nodes or _native()).packed_attention(q, k, v, tiles, packing.tokens, packing._longest, packing._pairs,
                                                  bool(causal), scale, stream)


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, *, base: float = 10000.0,
           dims: int | None = None, interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """q and k with the pairs of their features turned by position: pair i of a
    head by position * base^(-2i / dims). q is [..., heads, head_dim], k [...,
    kv_heads, head_dim], of one type (fp32, fp16 or bf16) on one GPU, positions
    [...] of int32 or int64. The first `dims` features (all, unless given) are
    paired i with i + dims/2, or 2i with 2i + 1 where `interleaved`; the others
    are copied. head_dim is at most 1024.

    Angles are formed in fp64; the arithmetic is fp32 and rounded once. Rows and
    heads may be strided. Differentiable once in q and k, backwards (a
    forward-mode tangent is refused); nothing but the positions is kept."""
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a tensor")
    dev = ops._device(q)
    ops.grad_code(q.dtype)
    if not isinstance(k, torch.Tensor) or k.dtype != q.dtype or k.device != dev:
        _refuse("k", k, q)
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be an int32 or int64 tensor")
    if positions.device != dev:
        raise ValueError(f"positions is on {positions.device}, expected {dev}")
    if q.dim() < 3 or k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"q and k must be [..., heads, head_dim], got {list(q.shape)} and {list(k.shape)}")
    if positions.shape != q.shape[:-2]:
        raise ValueError(f"positions must be {list(q.shape[:-2])}, got {list(positions.shape)}")
    heads, kv_heads, d = q.shape[-2], k.shape[-2], q.shape[-1]
    if not (1 <= heads <= MAX_HEADS and 1 <= kv_heads <= MAX_HEADS):
        raise ValueError(f"heads must lie in [1, {MAX_HEADS}], got {heads} and {kv_heads}")
    if not 1 <= d <= MAX_ROTARY_DIM:
        raise ValueError(f"head_dim must lie in [1, {MAX_ROTARY_DIM}], got {d}")
    dims = d if dims is None else int(dims)
    if dims % 2 or not 0 <= dims <= d:
        raise ValueError(f"dims must be even and at most head_dim, got {dims} of {d}")
    base = float(base)
    if not 0 < base < math.inf:
        raise ValueError(f"base must be positive and finite, got {base}")
    if positions.numel() > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} rows, got {positions.numel()}")
    flat = q.dim() == 3
    out = (_nodes or _native()).rotary(q if flat else q.reshape(-1, heads, d), k if flat else k.reshape(-1, kv_heads, d),
                                       positions.reshape(-1).contiguous(), base, dims, bool(interleaved),
                                       ops.stream_of(dev).value or 0)
    return out if flat else (out[0].view(q.shape), out[1].view(k.shape))


class AttentionBlock(torch.nn.Module):
    """Attention as one block of a stack: (hidden, normed, packing) -> (hidden,
    normed), beside GatedFFNBlock:

        q, k, v = normed Wq^T, normed Wk^T, normed Wv^T, q and k turned by position
        y       = packed_attention(q, k, v) Wo^T
        hidden  = hidden + branch_scale * gate * rms(y) * post_weight
        normed  = rms(hidden) * next_weight

    for normed [rows, width] whose first packing.tokens rows are the sequences.
    The four matrices are what Muon steps, the others vectors. The forward takes
    fp16 or bf16 parameters and inputs: give a dtype, or leave the cast to the
    engine's fp16 or bf16 mode."""

    def __init__(self, width: int, heads: int, kv_heads: int | None = None, head_dim: int | None = None, *,
                 causal: bool = True, rotary_base: float = 10000.0, branch_scale: float = 1.0, gate_init: float = 1.0,
                 eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"heads must be a multiple of kv_heads, got {heads} and {kv_heads}")
        if head_dim is None:
            if width % heads:
                raise ValueError(f"width {width} is not a multiple of {heads} heads: give head_dim")
            head_dim = width // heads
        if head_dim % 2 or not 2 <= head_dim <= MAX_HEAD_DIM:
            raise ValueError(f"head_dim must be even and at most {MAX_HEAD_DIM}, got {head_dim}")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.causal, self.rotary_base = bool(causal), float(rotary_base)
        self.branch_scale, self.eps = float(branch_scale), float(eps)
        kw = dict(device=device, dtype=dtype)

        def matrix(rows, cols):
            return torch.nn.Parameter(torch.empty(rows, cols, **kw).normal_(std=cols ** -0.5))

        self.w_q, self.w_k, self.w_v = (matrix(n * head_dim, width) for n in (heads, kv_heads, kv_heads))
        self.w_o = matrix(width, heads * head_dim)
        self.post_weight = torch.nn.Parameter(torch.ones(width, **kw))
        self.gate = torch.nn.Parameter(torch.full((width,), float(gate_init), **kw))
        self.next_weight = torch.nn.Parameter(torch.ones(width, **kw))

    def forward(self, hidden: torch.Tensor, normed: torch.Tensor, packing: PackedSequences
                ) -> tuple[torch.Tensor, torch.Tensor]:
        linear, rows = torch.nn.functional.linear, normed.shape[0]
        q = linear(normed, self.w_q).view(rows, self.heads, self.head_dim)
        k = linear(normed, self.w_k).view(rows, self.kv_heads, self.head_dim)
        v = linear(normed, self.w_v).view(rows, self.kv_heads, self.head_dim)
        positions = packing.positions
        if rows > packing.tokens:
            positions = torch.nn.functional.pad(positions, (0, rows - packing.tokens))
        q, k = rotary(q, k, positions, base=self.rotary_base)
        y = linear(packed_attention(q, k, v, packing, causal=self.causal).view(rows, -1), self.w_o)
        return gated_residual_norm(hidden, y, post_weight=self.post_weight, gate=self.gate,
                                   next_weight=self.next_weight, branch_scale=self.branch_scale, eps=self.eps)
