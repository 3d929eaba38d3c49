#!/usr/bin/env python3
"""A small tabular student that learns from a larger teacher's top logits.

Numerical columns go through ``CudaPiecewiseLinearEmbeddings``, categorical
ones through ``CudaCategoricalEmbeddings``; the features' embeddings are tokens
of a residual trunk whose blocks meet in ``CudaResidualNorm`` (the norm after a
block, its gate, the residual and the next block's norm in one pass), and
``CudaDistillationLoss`` compares the student with the teacher's top logits and
the labels.  Synthetic data; the teacher is a fixed random network, whose top
logits and log-sum are stored as a real one's would be.

    python examples/tabular_distillation.py [--device cuda] [--steps 60] [--autocast]

Prints the loss and the share of rows where the student agrees with the teacher.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from piecewiselinearembeddings_optimized_amd import (  # noqa: E402
    CudaCategoricalEmbeddings,
    CudaDistillationLoss,
    CudaPiecewiseLinearEmbeddings,
    CudaResidualNorm,
    compute_bins,
)


class Student(nn.Module):
    """Feature tokens [N, F, d], blocks that mix them, one linear head."""

    def __init__(self, bins, cardinalities, n_classes: int, d: int = 32, n_blocks: int = 2) -> None:
        super().__init__()
        f = len(bins) + len(cardinalities)
        self.numbers = CudaPiecewiseLinearEmbeddings(bins, d, activation=False, version="B")
        self.categories = CudaCategoricalEmbeddings(cardinalities, d)
        self.start = CudaResidualNorm(d, pre_norm="rms")
        # each block's end is the next one's beginning; the last one ends the trunk
        self.meet = nn.ModuleList(
            CudaResidualNorm(d, post_norm="rms", pre_norm="rms", gate="learned", gate_init=0.5) for _ in range(n_blocks))
        self.blocks = nn.ModuleList(nn.Sequential(nn.Linear(f * d, 4 * d), nn.GELU(), nn.Linear(4 * d, f * d))
                                    for _ in range(n_blocks))
        self.head = nn.Linear(f * d, n_classes)

    def forward(self, numbers, categories):
        stream = torch.cat([self.numbers(numbers), self.categories(categories).float()], dim=1)
        stream, normed = self.start(stream)
        for block, meet in zip(self.blocks, self.meet):
            branch = block(normed.flatten(1)).view(stream.shape)
            stream, normed = meet(stream, branch)
        return self.head(normed.flatten(1))


def make_data(n: int, n_numbers: int, cardinalities, n_classes: int, k: int, temperature: float, seed: int = 0):
    """Rows, labels, and a teacher's top logits with the log-sum over all classes."""
    gen = torch.Generator().manual_seed(seed)
    numbers = torch.randn(n, n_numbers, generator=gen)
    categories = torch.stack([torch.randint(0, c, (n,), generator=gen) for c in cardinalities], 1)
    categories[torch.rand(categories.shape, generator=gen) < 0.02] = -1          # missing values
    tables = [torch.randn(c + 1, 16, generator=gen) for c in cardinalities]
    hidden = torch.tanh(numbers @ torch.randn(n_numbers, 16, generator=gen))
    hidden = hidden + sum(t[col] for t, col in zip(tables, categories.T))
    logits = 2 * torch.tanh(hidden) @ torch.randn(16, n_classes, generator=gen)
    labels = torch.distributions.Categorical(logits=logits).sample()
    top, classes = logits.topk(k, dim=1)
    return numbers, categories, labels, top, classes, torch.logsumexp(logits / temperature, 1)


def train(device: str = "cuda", steps: int = 60, rows: int = 4096, batch: int = 512, autocast: bool = False,
          temperature: float = 2.0, report=print) -> list[float]:
    torch.manual_seed(0)
    cardinalities = [3, 40, 500]
    data = make_data(rows, 8, cardinalities, 100, 10, temperature)
    bins = compute_bins(data[0], n_bins=24)
    student = Student(bins, cardinalities, 100).to(device)
    loss_fn = CudaDistillationLoss(temperature, alpha=0.8)
    opt = torch.optim.AdamW(student.parameters(), lr=3e-3)
    data = [t.to(device) for t in data]
    losses = []
    for step in range(steps):
        at = slice(step * batch % rows, step * batch % rows + batch)
        numbers, categories, labels, top, classes, lse = (t[at] for t in data)
        with torch.autocast(device, dtype=torch.bfloat16, enabled=autocast):
            logits = student(numbers.contiguous(), categories)
        loss = loss_fn(logits, top, classes, lse, labels)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            agree = (logits.argmax(1) == classes[:, 0]).float().mean()
            report(f"step {step:3d}  loss {losses[-1]:.4f}  agrees with the teacher {float(agree):.3f}")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--autocast", action="store_true")
    args = ap.parse_args()
    train(args.device, args.steps, autocast=args.autocast)
