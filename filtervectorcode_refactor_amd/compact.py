"""Trains a narrow embedding on the exact neighbour lists of a base set.

The teacher is the build stage itself: the exact kNN lists of a group (ids, squared distances),
from the fp32 vectors.  The student maps the vectors to fewer dimensions by two matrices, one
for queries and one for the table, with every product in 8 bits; it is trained so that its
scores against the whole table give the teacher's lists (distillation at a temperature), and
its own first scores are compared with them.  Or it is trained against the nearest neighbour alone
(--loss nearest: cross entropy against the whole table, whose scores are then never in memory),
with the gradients scaled to a largest norm (--clip), and its lists are answered from a table in
8-bit whole numbers as well (--int8).

    python -m filtervectorcode_refactor_amd.compact --n 4000 --dim 128 --narrow 64 --steps 60
"""
from __future__ import annotations

import argparse
import time

import numpy as np
import torch

from . import scores
from .ung import HipContext


def vectors(n, dim, seed=0):
    """A seeded mixture: unit vectors around n / 100 centroids."""
    g = np.random.default_rng(seed)
    centres = g.standard_normal((max(n // 100, 1), dim))
    x = centres[g.integers(0, len(centres), n)] + 0.5 * g.standard_normal((n, dim))
    return (x / np.linalg.norm(x, axis=1, keepdims=True)).astype(np.float32)


def teacher_lists(X, k):
    """Exact neighbours of every vector among the others, as (ids, scores) on the GPU."""
    with HipContext(torch.cuda.current_device()) as ctx:
        ctx.prepare_vectors(X)
        ids, distances, _ = ctx.group_knn([0], [len(X)], k)
    ids, values = scores.entries_of_neighbors(ids, distances)
    return ids.cuda(), values.cuda()


def overlap(ids, wanted):
    """Mean share of each row of `wanted` that is in the same row of `ids`."""
    return (wanted[:, :, None] == ids[:, None, :]).any(2).float().mean().item()


class Student(torch.nn.Module):
    """Scores of every vector against the table of all, through `narrow` dimensions."""

    def __init__(self, dim, narrow):
        super().__init__()
        g = torch.Generator().manual_seed(1)
        start = torch.randn(narrow, dim, generator=g) / dim ** 0.5
        self.query = torch.nn.Parameter(start.clone().cuda())
        self.table = torch.nn.Parameter(start.clone().cuda())

    def embed(self, x):
        """The vectors' narrow embeddings as queries and as rows of the table."""
        return scores.linear_fp8(x, self.query), scores.linear_fp8(x, self.table)

    def forward(self, x):
        return without_own(scores.linear_fp8(*self.embed(x)))


def without_own(s):
    """Scores of all vectors against all, each one's own left out."""
    return s.masked_fill(torch.eye(len(s), dtype=torch.bool, device=s.device), -torch.inf)


def lists(student, x, k):
    """The student's first k of every vector."""
    with torch.no_grad():
        return scores.top_scores(student(x), k)[1]


def served_lists(student, x, k):
    """The same from a table in 8-bit whole numbers, as a program keeps it to answer queries."""
    with torch.no_grad():
        queries, table = student.embed(x)
        return scores.top_scores(without_own(scores.linear_int8(queries, *scores.quantize_int8(table))), k)[1]


def fit(X, k=32, narrow=64, steps=60, temperature=0.1, rate=0.02, loss="lists", clip=None):
    """(student, vectors on the GPU, the teacher's ids, losses of the steps, overlap before them)."""
    x = torch.from_numpy(X).cuda().bfloat16()
    ids, values = teacher_lists(X, k)
    nearest, own = ids[:, 0].contiguous(), torch.arange(len(X), dtype=torch.int32, device="cuda")
    student = Student(X.shape[1], narrow)
    optimizer = torch.optim.Adam(student.parameters(), lr=rate)
    before, losses = overlap(lists(student, x, k), ids), []
    for _ in range(steps):
        if loss == "nearest":
            rows = scores.table_loss(*student.embed(x), nearest, without=own, temperature=temperature)
        else:
            rows = scores.distill_loss(student(x), ids, values, temperature=temperature)
        mean = rows.mean()
        optimizer.zero_grad()
        mean.backward()
        if clip is not None:
            scores.clip_gradients([p.grad for p in student.parameters()], clip)
        optimizer.step()
        losses.append(mean.detach())
    return student, x, ids, [float(l) for l in losses], before


def train(X, k=32, narrow=64, steps=60, temperature=0.1, rate=0.02, loss="lists", clip=None):
    """(losses of the steps, overlap of the student's lists with the teacher's before and after)."""
    student, x, ids, losses, before = fit(X, k, narrow, steps, temperature, rate, loss, clip)
    return losses, before, overlap(lists(student, x, k), ids)


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("n", 4000), ("dim", 128), ("narrow", 64), ("k", 32), ("steps", 60)):
        parser.add_argument(f"--{name}", type=int, default=default)
    parser.add_argument("--temperature", type=float, default=0.1)
    parser.add_argument("--loss", choices=("lists", "nearest"), default="lists")
    parser.add_argument("--clip", type=float, default=None, help="largest norm of a step's gradients")
    parser.add_argument("--int8", action="store_true", help="lists from a table in 8-bit whole numbers too")
    a = parser.parse_args()
    X = vectors(a.n, a.dim)
    start = time.perf_counter()
    student, x, ids, losses, before = fit(X, a.k, a.narrow, a.steps, a.temperature, loss=a.loss, clip=a.clip)
    after = overlap(lists(student, x, a.k), ids)
    print(f"{a.steps} steps of {a.n} x {a.n} scores in {time.perf_counter() - start:.2f} s: "
          f"loss {losses[0]:.4f} -> {losses[-1]:.4f}, overlap with the exact {a.k} neighbours "
          f"{before:.3f} -> {after:.3f}")
    if a.int8:
        print(f"overlap of the lists from 8-bit whole numbers {overlap(served_lists(student, x, a.k), ids):.3f}")


if __name__ == "__main__":
    main()
