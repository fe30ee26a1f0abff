"""The forms of the sequence operators' kernels that large calls take, by their
sizes, at sizes as small as take them: the tolerances are those of
test_gpu_linear_cross_entropy and test_gpu_attention."""
from __future__ import annotations


import pytest

import test_gpu_attention as A
import test_gpu_linear_cross_entropy as C

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,d,vocab,dtype,reduction", [
    (2050, 2056, 2500, "bfloat16", "mean"),   # dx: 128-tiles
    (2100, 1030, 20001, "float16", "none"),   # dx: 128-tiles in three splits, of a copied weight
    (4099, 520, 70001, "bfloat16", "none"),   # the same of a vocabulary in two pieces, the second's sums on the first's
    (4101, 1032, 70001, "float16", "mean"),   # dx, dW and dz: 256-tiles, two pieces
    (4096, 1030, 70001, "bfloat16", "sum"),
])
def test_the_loss_in_large_tiles(gpu, tokens, d, vocab, dtype, reduction):
    x, w, targets, weights = C._make(tokens, d, vocab, dtype, seed=tokens + d, ignored=0.1)
    C._say(f"linear_cross_entropy {tokens} x {d} x {vocab} {dtype} {reduction}")
    C._check(C._run(x, w, targets, weights, reduction), x, w, targets, weights, reduction, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_long_sequences_with_many_blocks(gpu, causal, d, dtype):
    """704 blocks of 128 rows: one group of waves each, for sequences that few blocks
    would share between two."""
    A._compare([600, 700], 64, 16, d, dtype, causal, seed=d)


@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("lengths", [[512, 3], [577], [1000, 640]])
def test_few_blocks_in_bf16(gpu, lengths, d):
    """Two groups of waves: odd and even numbers of tiles, and a sequence of one."""
    A._compare(lengths, 3, 1, d, "bfloat16", len(lengths) == 1, seed=d)


@pytest.mark.parametrize("filler", [7.0, float("nan"), float("-inf")])
def test_padded_rows_of_a_block(gpu, filler):
    """Rows behind the sequences hold anything: AttentionBlock's results for the real
    rows are those of its operators on the same rows, to the bit, and of any other
    filler; a padded row's attention is zero, so that its hidden row stays as it was."""
    import torch
    from distributedspeed_amd import AttentionBlock, PackedSequences, gated_residual_norm, packed_attention, rotary
    torch.manual_seed(3)
    b = AttentionBlock(96, 4, 2, 32, gate_init=0.5, branch_scale=0.7, rotary_base=5e4, device="cuda", dtype=torch.bfloat16)
    packing = PackedSequences([33, 0, 90, 1])
    x = torch.randn(124, 96, device="cuda").bfloat16()

    def rows(value):
        return torch.cat((x, torch.full((6, 96), value, device="cuda").bfloat16()))

    zeros = rows(0.0)
    h0, n0 = b(zeros, zeros, packing)
    linear = torch.nn.functional.linear
    q, k, v = (linear(zeros, w).view(130, -1, 32) for w in (b.w_q, b.w_k, b.w_v))
    positions = torch.cat((packing.positions, torch.zeros(6, dtype=torch.int32, device="cuda")))
    q, k = rotary(q, k, positions, base=5e4)
    y = linear(packed_attention(q, k, v, packing).view(130, 128), b.w_o)
    assert not y[124:].any()
    h, n = gated_residual_norm(zeros, y, post_weight=b.post_weight, gate=b.gate, next_weight=b.next_weight, branch_scale=0.7)
    assert torch.equal(h0, h) and torch.equal(n0, n) and not h0[124:].any()
    more = rows(filler)
    h1, n1 = b(more, more, packing)
    assert torch.equal(h1[:124], h0[:124]) and torch.equal(n1[:124], n0[:124])
    assert torch.equal(h1[124:].nan_to_num(), more[124:].nan_to_num())


def test_a_step_of_the_example_changes_every_parameter(gpu):
    """Every parameter has a finite gradient and the two optimizers' steps move it."""
    import torch
    import test_gpu_sequence_use as U
    from distributedspeed_amd import AdamWOptimizer, MuonOptimizer, PackedSequences
    lm = U._example()
    torch.manual_seed(0)
    model = lm.PackedLM(256, 96, 4, 2, 2, device="cuda", dtype=torch.bfloat16)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    matrices = [p for n, p in model.named_parameters() if p.dim() == 2 and n != "embedding"]
    others = [p for n, p in model.named_parameters() if p.dim() != 2 or n == "embedding"]
    muon = MuonOptimizer(matrices, lr=0.02, weight_decay=0.0)
    adamw = AdamWOptimizer(others, lr=3e-2, weight_decay=0.0, param_dtype=torch.bfloat16)
    tokens, targets, lengths = lm.batch(256, 512, torch.Generator().manual_seed(0))
    model(tokens.cuda(), targets.cuda(), PackedSequences(lengths)).backward()
    assert all(p.grad.isfinite().all() and p.grad.any() for p in model.parameters())
    muon.step()
    adamw.step()
    for n, p in model.named_parameters():
        assert p.isfinite().all() and not torch.equal(p, before[n]), n


def test_attention_past_its_limits_is_refused(gpu):
    """By the wrapper, as its other arguments: a scale that fp32 does not hold, and more
    tiles and heads than a launch takes."""
    import torch
    from distributedspeed_amd import PackedSequences, packed_attention
    q = torch.zeros(4, 2, 8, device="cuda").bfloat16()
    for scale in (1e-50, 2.0 ** -127, 2e38, float("inf"), -1.0):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(q, q, q, PackedSequences([4]), scale=scale)
    assert packed_attention(q, q, q, PackedSequences([4]), scale=2.0 ** -126).isfinite().all()
    one = torch.zeros(1, 1, 8, device="cuda").bfloat16()
    n = 1 << 14
    with pytest.raises(ValueError, match="tiles"):
        packed_attention(one.expand(n, 1024, 8), one.expand(n, 1, 8), one.expand(n, 1, 8), PackedSequences([1] * n))
