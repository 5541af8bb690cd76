"""GPU tests of the distillation's listed columns where the teacher's remaining mass stands against
little of the student's: every column by the error of the terms that it has, in 64 bits."""
import math

import numpy as np
import pytest
import torch

from filtervectorcode_refactor_amd import scores as S

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"fp32": 2.0 ** -126, "fp16": 2.0 ** -25, "bf16": 2.0 ** -126}
EPS = 2.0 ** -23


def _exact(x, ids, val, lse, w, t):
    """Of one row: loss, gradient, and each column's sum of magnitudes (1 + |exponent|) over the
    terms W q_j, p_j and p_r q_j / Q_r that it has."""
    z = x.astype(np.float64) / t
    there = (ids >= 0) & (ids < len(x)) & (val != -np.inf)
    at, a = ids[there], val[there].astype(np.float64) / t
    m = z.max()
    q = np.exp(z - m)
    log_total = math.log(q.sum())
    q /= q.sum()
    listed = np.zeros(len(x), bool)
    listed[at] = True
    p = np.exp(a - float(lse))
    rest = max(0.0, 1 - p.sum())
    rest_top = z[~listed].max() if (~listed).any() else -np.inf
    log_rest = -np.inf if rest_top == -np.inf else rest_top + math.log(np.exp(z[~listed] - rest_top).sum()) - m - log_total
    if log_rest == -np.inf:
        rest = 0.0
    loss = (p * ((a - float(lse)) - (z[at] - m - log_total))).sum()
    if rest > 0:
        loss += rest * (math.log(rest) - log_rest)
    dense, far = np.zeros(len(x)), np.zeros(len(x))
    np.add.at(dense, at, p)
    np.add.at(far, at, p * (2 + np.abs(a) + abs(float(lse))))
    share = np.where(listed, 0.0, np.exp(np.where(listed, -np.inf, z - m - log_total - log_rest if rest > 0 else -np.inf)))
    mass = p.sum() + rest
    grad = (mass * q - dense - rest * share) * w / t
    size = 1 + np.minimum(np.where(np.isfinite(z), np.abs(z - m), 0), 200)
    # p_r is 1 less a sum: off by that sum's rounding whatever its size; W = 1 or sum p_k, as that
    scale = (q * size * mass + far + (share * size if rest > 0 else 0.0)) * abs(w) / t
    return loss, grad, scale, listed


def _check(x, kind, ids, val, lse, t):
    """Every term of a gradient passes at most depth + 8 operations of 32 bits that scale with it
    (the sum over the row, its own exponential by its exponent, the products)."""
    n, v = x.shape
    w = np.random.default_rng(n + v).random(n).astype(np.float32) + 0.5
    view = torch.from_numpy(x).to(TYPES[kind]).cuda()
    x = view.float().cpu().numpy()
    args = [torch.from_numpy(a).cuda() for a in (ids, val)]
    t_lse, tw = torch.from_numpy(lse).cuda(), torch.from_numpy(w).cuda()
    loss, grad = S.distill_step(view, *args, tw, teacher_lse=t_lse, temperature=t)
    loss2, saved = S.distill_forward(view, *args, teacher_lse=t_lse, temperature=t)
    grad2 = S.distill_backward(tw, view, *args, saved, temperature=t)
    depth = 2 * math.log(v + 1) + v / 256 + 100
    near = math.inf
    for r in range(n):
        want_loss, want, scale, listed = _exact(x[r], ids[r], val[r], lse[r], float(w[r]), t)
        size = np.abs(x[r][np.isfinite(x[r])]).max() / t + 20
        for got in (loss, loss2):
            assert abs(float(got[r]) - want_loss) <= EPS * (depth + 8 * size) * 2, (r, float(got[r]), want_loss)
        bound = EPS * (depth + 8) * scale + HALF_ULP[kind] * 1.001 * np.abs(want) + TINY[kind]
        for got in (grad, grad2):
            err = np.abs(got[r].float().cpu().numpy().astype(np.float64) - want)
            assert (err <= bound).all(), (r, np.argwhere(err > bound)[:4], (err / bound).max())
        near = min(near, (EPS * (depth + 8) * scale / np.maximum(np.abs(want), 1e-30))[listed].min())
    assert near < 1  # bounds above every listed column's gradient would say nothing


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("v", [64, 5000, 70_000])
@pytest.mark.parametrize("gap", [0.0, 3.0, 12.0, 40.0, 110.0])
def test_listed_columns_above_the_rest(v, gap, kind):
    """The listed scores lie `gap` above all others: the student's mass outside the list falls from
    most of it to 1e-46."""
    g = np.random.default_rng(v + int(gap))
    n, k = 6, 8
    x = g.standard_normal((n, v)).astype(np.float32) - (20.0 if gap > 60 else 0.0)
    ids = np.stack([g.choice(v, k, replace=False) for _ in range(n)]).astype(np.int32)
    val = (g.standard_normal((n, k)) * 1.5 + 2).astype(np.float32)
    for r in range(n):
        x[r, ids[r]] += np.float32(gap)
    ids[1, 3:] = -1
    val[2, 5:] = -np.inf
    for t in (1.0, 2.0):
        there = (ids >= 0) & (val > -np.inf)
        mass = np.where(there, np.exp(val.astype(np.float64) / t), 0).sum(axis=1)
        for more in (0.7, 1e-3):  # of the teacher's mass outside its list, and nearly none
            _check(x, kind, ids, val, np.log(mass * (1 + more)).astype(np.float32), t)


@pytest.mark.parametrize("v", [64, 70_000])
def test_one_listed_column_with_all_of_the_students_mass(v):
    x = np.full((4, v), -80.0, np.float32)
    ids, val = np.full((4, 4), -1, np.int32), np.full((4, 4), -np.inf, np.float32)
    ids[:, 0], val[:, 0] = 5, 1.0
    x[:, 5] = [30.0, 0.0, -60.0, -79.0]
    lse = np.log(np.exp(np.float64(1.0)) + np.array([0.7, 0.7, 1e-3, 20.0])).astype(np.float32)
    _check(x, "fp32", ids, val, lse, 1.0)
