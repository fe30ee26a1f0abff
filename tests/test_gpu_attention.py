"""packed_attention and its gradients on the GPU against the formulas in 64 bits.

Tolerances, element by element, from what is rounded. u is half a step of the
type (2^-8 for bf16, 2^-11 for fp16); P is rounded once (to u of itself) before it
meets v or do, dS once before it meets k or q, and each result once:

  |out - o| <= u (|o| + P |v|),            |dv| <= u (|dv| + P^T |do|)
  |dq| <= u (|dq| + scale M |k|),          |dk| <= u (|dk| + scale M^T |q|)

with M = |dS| + P E: dS = P (dP - delta) takes delta = do o from the output as it
was summed (before its own rounding, which is kept beside it), whose P had been
rounded, so that |o~ - o| <= u P |v| and delta is off by up to u E, E = |do| (P |v|)
of the query's row. What fp32 adds (scores, exponentials, sums, delta from an output held twice) is
within 2^-13 of the sums of magnitudes P |v|, P^T |do|, and, with D = P (|do| |v|
+ |do| |o|), scale D |k| and scale D^T |q|."""
from __future__ import annotations

import math
import sys

import pytest

pytestmark = pytest.mark.gpu

U = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
FP32 = 2.0 ** -13
LEAST = {"bfloat16": 0.0, "float16": 2.0 ** -25}  # below 2^-14 fp16's step is 2^-24 whatever the value: half of it


def _say(msg):
    print(f"[gpu-test] {msg}", file=sys.stderr, flush=True)


def _make(rows, heads, kv_heads, d, dtype, seed=0, sharp=1.5, dout=0.3):
    import torch
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = getattr(torch, dtype)

    def normal(*s, std=1.0):
        return (torch.randn(*s, generator=gen, device="cuda") * std).to(dt)

    return (normal(rows, heads, d, std=sharp), normal(rows, kv_heads, d), normal(rows, kv_heads, d),
            normal(rows, heads, d, std=dout))


def _exact(q, k, v, do, lengths, causal, scale):
    """Results and, for each, what its rounding errors are in proportion to and
    what fp32's are."""
    import torch
    group = q.shape[1] // k.shape[1]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    names = {"out": q, "dq": q, "dk": k, "dv": v}
    want, mags, sums = ({n: torch.zeros_like(t) for n, t in names.items()} for _ in range(3))
    first = 0
    for n in lengths:
        at = slice(first, first + n)
        first += n
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        for h in range(q.shape[1]):
            g = h // group
            qq, kk, vv, dd = q[at, h], k[at, g], v[at, g], do[at, h]
            s = (qq @ kk.t()) * scale
            p = torch.softmax(s.masked_fill(hidden, -math.inf) if causal else s, 1)
            o = p @ vv
            dp = dd @ vv.t()
            ds = p * (dp - (dd * o).sum(1, keepdim=True)) * scale
            off = p * (dd.abs() * (p @ vv.abs())).sum(1, keepdim=True) * scale  # P E
            loose = p * (dd.abs() @ vv.abs().t() + (dd.abs() * o.abs()).sum(1, keepdim=True)) * scale
            want["out"][at, h] = o
            want["dq"][at, h] = ds @ kk
            want["dk"][at, g] += ds.t() @ qq
            want["dv"][at, g] += p.t() @ dd
            mags["out"][at, h] = p @ vv.abs()
            mags["dq"][at, h] = (ds.abs() + off) @ kk.abs()
            mags["dk"][at, g] += (ds.abs() + off).t() @ qq.abs()
            mags["dv"][at, g] += p.t() @ dd.abs()
            sums["out"][at, h] = mags["out"][at, h]
            sums["dq"][at, h] = loose @ kk.abs()
            sums["dk"][at, g] += loose.t() @ qq.abs()
            sums["dv"][at, g] += p.t() @ dd.abs()
    return want, mags, sums


def _run(q, k, v, do, lengths, causal=True, scale=None):
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention
    args = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*args, PackedSequences(lengths), causal=causal, scale=scale)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, args, do))))


def _check(got, exact, dtype):
    want, mags, sums = exact
    u = U[dtype]
    for name, g in got.items():
        w = want[name]
        assert g.shape == w.shape and bool(g.isfinite().all()), name
        bound = u * (1 + u) * (w.abs() + mags[name]) + FP32 * sums[name] + 2.0 ** -24 * w.abs().max() + LEAST[dtype]
        far = ((g.double() - w).abs() - bound).max().item() if w.numel() else 0
        assert far <= 0, (name, far)


def _compare(lengths, heads, kv_heads, d, dtype, causal, seed=0, **kw):
    args = _make(sum(lengths), heads, kv_heads, d, dtype, seed, **kw)
    _say(f"attention {lengths} {heads}/{kv_heads} x {d} {dtype} {'causal' if causal else 'full'}")
    _check(_run(*args, lengths, causal), _exact(*args, lengths, causal, 1 / math.sqrt(d)), dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", [[1], [2], [17], [31, 32, 33], [63, 64, 65], [127, 128, 129], [1, 1, 0, 2, 1],
                                     [257, 300], [0, 513, 0, 1, 190], [1001]])
def test_lengths(gpu, lengths, causal, dtype):
    _compare(lengths, 2, 1, 64, dtype, causal, seed=sum(lengths))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [1, 5, 8, 16, 24, 40, 65, 72, 80, 100, 128, 136, 160, 255, 256])
def test_head_sizes(gpu, d, causal):
    """Every padded size, features that are no multiple of eight among them."""
    _compare([70, 130, 1, 300], 2, 2, d, "bfloat16", causal, seed=d)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (8, 8), (9, 3), (12, 2), (32, 8)])
def test_head_layouts(gpu, heads, kv_heads):
    _compare([200, 77, 260], heads, kv_heads, 64, "float16", True, seed=heads)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_work_in_parts(gpu, d, causal):
    """One key head and a long sequence: the keys' gradients come in parts that
    end inside a head, and are joined."""
    _compare([1500, 3, 700], 3, 1, d, "bfloat16", causal, seed=d)


@pytest.mark.parametrize("d", [32, 96, 192])
@pytest.mark.parametrize("causal", [True, False])
def test_sizes_between_in_parts(gpu, d, causal):
    _compare([700, 1, 555], 4, 2, d, "bfloat16", causal)


@pytest.mark.parametrize("d", [64, 128])
def test_scores_below_the_range_of_fp32(gpu, d):
    """Keys whose scores are -inf in fp32 have no weight, also where a row's first
    tiles hold no others."""
    lengths = [150, 20]
    q, k, v, do = _make(170, 4, 2, d, "bfloat16")
    q[..., 0] = 2.0 ** 70
    k[..., 0] = 0
    k[:70, :, 0] = -2.0 ** 70
    _check(_run(q, k, v, do, lengths, False), _exact(q, k, v, do, lengths, False, 1 / math.sqrt(d)), "bfloat16")


@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("lengths", [[511], [512], [513, 1], [575], [576, 2], [577], [640, 0, 1000]])
def test_few_blocks(gpu, lengths, d):
    """From 512 rows on, where there are few blocks, two groups of waves share one's
    tiles: even and odd numbers of them, and other sequences of one tile."""
    _compare(lengths, 3, 1, d, "float16", len(lengths) != 2)


def test_a_given_scale(gpu):
    args = _make(300, 2, 2, 64, "bfloat16", 3)
    _check(_run(*args, [300], True, 0.4), _exact(*args, [300], True, 0.4), "bfloat16")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("sharp,dout", [(30.0, 0.3), (1.0, 1e-4), (1.0, 300.0), (0.0, 1.0)])
def test_saturated_rows_and_gradients_of_any_scale(gpu, sharp, dout, dtype):
    """Scores of hundreds (P is zero or one nearly everywhere), none at all, and
    output gradients whose products leave fp16's range unless scaled. Where they
    are small the results themselves come near fp16's least step, 2^-25 at most."""
    lengths = [5, 400]
    args = _make(405, 2, 1, 64, dtype, 7, sharp=sharp, dout=dout)
    want, mags, sums = _exact(*args, lengths, True, 0.125)
    got = _run(*args, lengths, True, 0.125)
    # scores of magnitude s have fp32 errors of 2^-24 s a term: P's grow with them
    grow = max(1.0, sharp)
    step = 2.0 ** -25 if dtype == "float16" else 0.0
    for name, g in got.items():
        bound = (U[dtype] * 1.01 * (want[name].abs() + mags[name]) + grow * FP32 * sums[name]
                 + 2.0 ** -24 * want[name].abs().max() + step)
        assert bool(g.isfinite().all()), name
        assert ((g.double() - want[name]).abs() <= bound).all(), name


def test_one_key_rows(gpu):
    """P is one whatever the score: dq and dk are zero, not rounding errors, the
    output is v and dv is the output's gradient."""
    import torch
    q, k, v, do = _make(50, 2, 2, 64, "bfloat16", 1)
    got = _run(q, k, v, do, [1] * 50, True)
    assert not got["dq"].any() and not got["dk"].any()
    assert torch.equal(got["out"], v) and torch.equal(got["dv"], do)
    assert not _run(q, k, v, do, [1] * 50, False)["dq"].any()


@pytest.mark.parametrize("causal", [True, False])
def test_gradients_against_differences(gpu, causal):
    """Along a random direction, against central differences of the exact output
    (their own error is of the order of 1e-6 here)."""
    import torch
    lengths, scale = [90, 7], 1 / math.sqrt(40)
    q, k, v, do = _make(97, 4, 2, 40, "bfloat16", 11)
    got = _run(q, k, v, do, lengths, causal)
    want, mags, sums = _exact(q, k, v, do, lengths, causal, scale)
    gen = torch.Generator("cuda").manual_seed(5)
    h = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(*(q, k, v)[i].shape, generator=gen, device="cuda", dtype=torch.float64)

        def loss(sign):
            moved = [t.double() for t in (q, k, v)]
            moved[i] = moved[i] + sign * h * way
            return (_exact(*moved, do, lengths, causal, scale)[0]["out"] * do.double()).sum()

        change = (loss(1) - loss(-1)) / (2 * h)
        u = U["bfloat16"]
        slack = ((u * 1.01 * (want[name].abs() + mags[name]) + FP32 * sums[name]) * way.abs()).sum() + 1e-4
        assert abs((got[name].double() * way).sum() - change) <= slack, name


def _layouts(t):
    """The same values laid out otherwise: parts of wider rows, heads outermost, an
    odd address, an odd row stride, features apart, and backwards."""
    import torch
    n, h, d = t.shape
    wide = torch.full((n, h + 3, d), float("nan"), dtype=t.dtype, device=t.device)
    wide[:, 2:2 + h] = t
    yield "parts of wider rows", wide[:, 2:2 + h]
    outer = torch.empty(h, n, d, dtype=t.dtype, device=t.device)
    outer.copy_(t.transpose(0, 1))
    yield "heads outermost", outer.transpose(0, 1)
    odd = torch.empty(n * h * d + 3, dtype=t.dtype, device=t.device)[3:].view(n, h, d)
    odd.copy_(t)
    yield "an odd address", odd
    rows = torch.full((n, h * d + 5), float("nan"), dtype=t.dtype, device=t.device)
    rows[:, :h * d] = t.reshape(n, -1)
    yield "an odd row stride", rows[:, :h * d].unflatten(1, (h, d))
    apart = torch.full((n, h, d, 2), float("nan"), dtype=t.dtype, device=t.device)
    apart[..., 0] = t
    yield "features apart", apart[..., 0]


def test_layouts(gpu):
    """To the bit what contiguous tensors give, gradients of such outputs too."""
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention
    lengths = [150, 1, 60]
    q, k, v, do = _make(211, 4, 2, 72, "bfloat16", 2)
    plain = _run(q, k, v, do, lengths)
    packing = PackedSequences(lengths)
    for (name, a), (_, b), (_, c), (_, e) in zip(_layouts(q), _layouts(k), _layouts(v), _layouts(do)):
        _say(name)
        args = [t.detach().requires_grad_(True) for t in (a, b, c)]
        out = packed_attention(*args, packing)
        got = dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, args, e))))
        assert all(torch.equal(got[x], plain[x]) for x in plain), name
    # a key head that all query heads share by expansion, and a summed output
    one = k[:, :1].expand(-1, 4, -1)
    same = packed_attention(q, one, v[:, :1].expand(-1, 4, -1), packing)
    assert torch.equal(same, packed_attention(q, k[:, :1], v[:, :1], packing))
    x = q.clone().requires_grad_(True)
    g, = torch.autograd.grad(packed_attention(x, k, v, packing).sum(), x)
    assert torch.equal(g, _run(q, k, v, torch.ones_like(do), lengths)["dq"])


def test_rows_past_32_bits(gpu):
    """Rows 65536 elements apart, whose last lie beyond 2^31 elements."""
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention
    rows, stride = 33000, 65536
    buf = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
    lengths = [100] * 330
    q, k, v, do = _make(rows, 2, 1, 64, "bfloat16", 4)
    view = buf.view(rows, stride)
    view[:, :128] = q.view(rows, 128)
    view[:, 1024:1088] = k[:, 0]
    view[:, 2048:2112] = v[:, 0]
    view[:, 4096:4224] = do.view(rows, 128)
    parts = [view[:, :128].unflatten(1, (2, 64)), view[:, 1024:1088][:, None], view[:, 2048:2112][:, None]]
    plain = _run(q, k, v, do, lengths)
    args = [t.detach().requires_grad_(True) for t in parts]
    out = packed_attention(*args, PackedSequences(lengths))
    got = torch.autograd.grad(out, args, view[:, 4096:4224].unflatten(1, (2, 64)))
    assert torch.equal(out, plain["out"])
    assert all(torch.equal(a, plain[n]) for a, n in zip(got, ("dq", "dk", "dv")))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_what_is_not_finite_stays_in_its_sequence(gpu, value, dtype):
    """Beside a spoilt sequence, and before rows behind the last one that hold
    anything, every other row is what it is without them, to the bit (for the
    gradients in fp16: without the spoilt sequence's share in their scale, which a
    spoilt row has no part in)."""
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention
    lengths, rows = [40, 100, 7, 130], 300
    q, k, v, do = _make(rows, 4, 2, 64, dtype, 8)
    packing = PackedSequences(lengths)

    def run(q, k, v, do):
        args = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = packed_attention(*args, packing)
        return (out.detach(), *torch.autograd.grad(out, args, do))

    clean = run(q, k, v, do)
    bad = [t.clone() for t in (q, k, v, do)]
    for t in bad:
        t[277:] = value
    for a, b in zip(run(*bad), clean):
        assert torch.equal(a[:277], b[:277]) and not a[277:].any()
    for i in range(3):
        bad = [t.clone() for t in (q, k, v, do)]
        bad[i][60, 0, 3] = value  # in the second sequence
        for a, b in zip(run(*bad), clean):
            assert torch.equal(a[:40], b[:40]) and torch.equal(a[140:277], b[140:277])
        assert not run(*bad)[0][60:140].isfinite().all()


def test_a_sequence_does_not_depend_on_the_packing(gpu):
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention
    lengths = [333, 64, 1, 200]
    q, k, v, _ = _make(sum(lengths), 4, 2, 64, "bfloat16", 9)
    whole = packed_attention(q, k, v, PackedSequences(lengths))
    first = 0
    for n in lengths:
        at = slice(first, first + n)
        first += n
        assert torch.equal(whole[at], packed_attention(q[at], k[at], v[at], PackedSequences([n])))


def test_results_repeat(gpu):
    import torch
    args = _make(3000, 8, 2, 128, "bfloat16", 10)
    a, b = (_run(*args, [2000, 1000]) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_only_the_gradients_that_are_wanted(gpu):
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention
    q, k, v, do = _make(150, 2, 2, 64, "bfloat16", 12)
    packing = PackedSequences([150])
    full = _run(q, k, v, do, [150])
    for i, name in enumerate(("dq", "dk", "dv")):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        out = packed_attention(*args, packing)
        g, = torch.autograd.grad(out, args[i], do)
        assert torch.equal(g, full[name])


def test_no_rows(gpu):
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention
    for lengths, rows in (([], 0), ([0, 0], 0), ([], 5), ([0], 5)):
        args = [torch.randn(rows, h, 64, device="cuda").bfloat16().requires_grad_(True) for h in (4, 2, 2)]
        packing = PackedSequences(lengths)
        assert packing.tokens == 0 and packing.positions.shape == (0,)
        out = packed_attention(*args, packing)
        assert out.shape == (rows, 4, 64) and not out.any()
        out.sum().backward()
        assert all(t.grad.shape == t.shape and not t.grad.any() for t in args)
