"""Trains a small causal language model on packed sequences of different lengths:
blocks of attention and of gated feed-forward layers, with the cross entropy taken
straight from the hidden rows. Muon steps the blocks' matrices, AdamW the rest.

The task: each sequence repeats a short random phrase, so that a model that looks
back far enough can predict its tokens.

    python examples/train_packed_lm.py [--width 256] [--heads 4] [--kv-heads 2] [--blocks 2] [--vocab 512]
                                       [--tokens 2048] [--steps 60]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from distributedspeed_amd import (AdamWOptimizer, AttentionBlock, GatedFFNBlock, MuonOptimizer,  # noqa: E402
                                  PackedSequences, gated_residual_norm, linear_cross_entropy)

IGNORE = -100


class PackedLM(torch.nn.Module):
    def __init__(self, vocab: int, width: int, heads: int, kv_heads: int, blocks: int, **kw):
        super().__init__()
        self.embedding = torch.nn.Parameter(torch.empty(vocab, width, **kw).normal_(std=width ** -0.5))
        self.first_weight = torch.nn.Parameter(torch.ones(width, **kw))
        self.attention = torch.nn.ModuleList(AttentionBlock(width, heads, kv_heads, gate_init=0.5, **kw)
                                             for _ in range(blocks))
        self.ffn = torch.nn.ModuleList(GatedFFNBlock(width, 8 * width // 3 // 8 * 8, gate_init=0.5, **kw)
                                       for _ in range(blocks))

    def forward(self, tokens: torch.Tensor, targets: torch.Tensor, packing: PackedSequences) -> torch.Tensor:
        """The mean loss over the targets that are not IGNORE."""
        x = torch.nn.functional.embedding(tokens, self.embedding)
        hidden, normed = gated_residual_norm(x, next_weight=self.first_weight)
        for attention, ffn in zip(self.attention, self.ffn):
            hidden, normed = attention(hidden, normed, packing)
            hidden, normed = ffn(hidden, normed)
        return linear_cross_entropy(normed, self.embedding, targets, ignore_index=IGNORE)


def batch(vocab: int, tokens: int, gen: torch.Generator) -> tuple[torch.Tensor, torch.Tensor, list[int]]:
    """Tokens, targets (the next token; none behind a sequence's last) and the
    sequences' lengths, which add up to `tokens`."""
    lengths, rows, targets = [], [], []
    while sum(lengths) < tokens:
        n = min(int(torch.randint(16, 300, (), generator=gen)), tokens - sum(lengths))
        period = int(torch.randint(3, 12, (), generator=gen))
        row = torch.randint(0, vocab, (period,), generator=gen).repeat(n // period + 1)[:n]
        lengths.append(n)
        rows.append(row)
        targets.append(torch.cat((row[1:], torch.tensor([IGNORE]))))
    return torch.cat(rows), torch.cat(targets), lengths


def train(vocab: int, width: int, heads: int, kv_heads: int, blocks: int, tokens: int, steps: int, seed: int = 0
          ) -> list[float]:
    """The loss of every step."""
    device = torch.device("cuda", 0)
    torch.manual_seed(seed)
    gen = torch.Generator().manual_seed(seed)
    model = PackedLM(vocab, width, heads, kv_heads, blocks, device=device, dtype=torch.bfloat16)
    matrices = [p for n, p in model.named_parameters() if p.dim() == 2 and n != "embedding"]
    others = [p for n, p in model.named_parameters() if p.dim() != 2 or n == "embedding"]
    muon = MuonOptimizer(matrices, lr=0.02, weight_decay=0.0)
    adamw = AdamWOptimizer(others, lr=3e-3, weight_decay=0.0, param_dtype=torch.bfloat16)
    losses = []
    for _ in range(steps):
        rows, targets, lengths = batch(vocab, tokens, gen)
        loss = model(rows.to(device), targets.to(device), PackedSequences(lengths, device=device))
        loss.backward()
        muon.step()
        adamw.step()
        muon.zero_grad()
        adamw.zero_grad()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("vocab", 512), ("width", 256), ("heads", 4), ("kv-heads", 2), ("blocks", 2), ("tokens", 2048),
                        ("steps", 60)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args()
    losses = train(a.vocab, a.width, a.heads, a.kv_heads, a.blocks, a.tokens, a.steps)
    for i in range(0, len(losses), max(1, len(losses) // 8)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"step {len(losses) - 1:4d}  loss {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
