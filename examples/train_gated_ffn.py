"""Trains a stack of gated feed-forward blocks on a synthetic regression task:
Muon steps the blocks' matrices, AdamW their vectors.

    python examples/train_gated_ffn.py [--width 256] [--inner 688] [--blocks 4] [--tokens 512] [--steps 40]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from distributedspeed_amd import AdamWOptimizer, GatedFFNBlock, MuonOptimizer, gated_residual_norm  # noqa: E402


class Stack(torch.nn.Module):
    def __init__(self, width: int, inner: int, blocks: int, **kw):
        super().__init__()
        self.first_weight = torch.nn.Parameter(torch.ones(width, **kw))
        self.blocks = torch.nn.ModuleList(GatedFFNBlock(width, inner, gate_init=0.5, **kw) for _ in range(blocks))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        hidden, normed = gated_residual_norm(x, next_weight=self.first_weight)
        for block in self.blocks:
            hidden, normed = block(hidden, normed)
        return normed


def train(width: int, inner: int, blocks: int, tokens: int, steps: int, seed: int = 0) -> list[float]:
    """The loss of every step."""
    device = torch.device("cuda", 0)
    torch.manual_seed(seed)
    model = Stack(width, inner, blocks, device=device, dtype=torch.bfloat16)
    target = torch.randn(width, width, device=device) / width ** 0.5
    matrices = [p for p in model.parameters() if p.dim() == 2]
    vectors = [p for p in model.parameters() if p.dim() == 1]
    muon = MuonOptimizer(matrices, lr=0.02, weight_decay=0.0)
    adamw = AdamWOptimizer(vectors, lr=1e-3, weight_decay=0.0, param_dtype=torch.bfloat16)
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, width, device=device, dtype=torch.bfloat16)
        want = torch.tanh(x.float() @ target)
        loss = (model(x).float() - want).square().mean()
        loss.backward()
        muon.step()
        adamw.step()
        muon.zero_grad()
        adamw.zero_grad()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("width", 256), ("inner", 688), ("blocks", 4), ("tokens", 512), ("steps", 40)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args()
    losses = train(a.width, a.inner, a.blocks, a.tokens, a.steps)
    for i in range(0, len(losses), max(1, len(losses) // 8)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"step {len(losses) - 1:4d}  loss {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
