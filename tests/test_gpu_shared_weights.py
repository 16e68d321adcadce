"""The bits of a weight in the shared read: one query's are multiplied by V in 16 bits, a chunk's in 8.

One-query reads multiply V by a weight's bf16 rounding and by that rounding's rest in bf16, which leaves 2^-8 of 2^-8 of the weight: 2^-16 of
it at most. With A = sum_j w_j |v_j| and S the largest |score| (log2), an output is off by 2^-8 of itself (its own rounding) and by A times
2^-16 and, twice, what exponents and sums take: 2^-17 + (S + 8) 2^-20.
"""
from __future__ import annotations

import math

import pytest
import torch

from attention_lab import shared_prefix_attention
from attention_lab.hip_attend import attend_paged
from test_gpu_shared import CASES, LOG2E, Case, make

pytestmark = pytest.mark.gpu


def near(got, want, size, scores):
    err = 2.0 ** -8 * want.abs() + size * (2.0 ** -16 + 2 * (2.0 ** -17 + (scores.abs().max() * LOG2E + 8) * 2.0 ** -20))
    return ((got - want).abs() <= err).all(), ((got - want).abs() / err).max()


@pytest.mark.parametrize("name", [n for n, c in CASES.items() if c[-1] == 1])
def test_cases(gpu, name):
    """Every one-query case, with the bound of 16-bit weights."""
    c = make(name, 4)
    got = c.call(gpu).double().cpu()
    for i in range(len(c.lengths)):
        at = list(c.legal(i))
        if not at:
            assert (got[i] == 0).all()
            continue
        _, p, r = (torch.tensor(x) for x in zip(*at))
        k, v = (x[p, :, r].double().transpose(0, 1) for x in (c.k, c.v))
        s = c.q[i, :, :, 0].double() @ k.transpose(1, 2) / 128 ** 0.5
        w = torch.softmax(s, dim=-1)
        fine, worst = near(got[i, :, :, 0], w @ v, w @ v.abs(), s)
        assert fine, (i, worst)


@pytest.mark.parametrize("n,prefix,h,page,partitions", [
    (1, 0, 1, 16, None), (1, 0, 16, 64, (0, 3)), (3, 1024, 2, 64, None), (3, 1024, 2, 64, (4, 2)), (40, 1024, 4, 32, None),
    (5, 512, 3, 4, None), (40, 512, 4, 2, None),
])
def test_roundings_that_add_up(gpu, n, prefix, h, page, partitions):
    """A third of the keys weigh 1 and have v = 1; the others weigh (1 + 2^-8 - 2^-12) / 2 and have v = -1. Rounded to bf16 every one of
    those is off by 2^-8 the same way, and the output, about -2^-9, by as much as itself."""
    weight = 0.5 * (1 + 2.0 ** -8 - 2.0 ** -12)
    keys = 1536
    c = Case(3, [n], [prefix], [keys] * n, page, 1, h, 1)
    heavy = torch.arange(keys) % 3 == 0
    for i in range(n):
        for j, p, r in c.legal(i):
            c.k[p, 0, r] = 0
            c.k[p, 0, r, 0] = 0.0 if heavy[j] else -1.0
            c.v[p, 0, r] = 1.0 if heavy[j] else -1.0
    c.q.zero_()
    c.q[..., 0] = 1
    scale = -math.log(weight)
    got = c.call(gpu, scale=scale, partitions=partitions).double().cpu()
    w = torch.where(heavy, 1.0, math.exp(-torch.tensor(scale, dtype=torch.float32).double().item())).double()
    w /= w.sum()
    want = (w * torch.where(heavy, 1.0, -1.0)).sum()
    fine, worst = near(got, want, torch.tensor(1.0, dtype=torch.float64), torch.tensor(scale))
    assert fine, (got.flatten()[:4], want, worst)
    if h > 8:   # the paged read's most
        return
    q, k, v, table, *_ = c.args(gpu)
    other = attend_paged(q[:, :, :, 0], k, v, table, length=keys, scale=scale, out_dtype=torch.float32).double().cpu()
    assert (got[:, :, :, 0] - other).abs().max() <= 2.0 ** -8 * abs(want) + 2.0 ** -13   # the two reads' sums


def test_chunks_round_once(gpu):
    """The same in a chunk: the documented 2^-8 of each weight."""
    for name in ("chunk_17", "chunk_runs"):
        c = make(name, 4)
        c.check(shared_prefix_attention(*c.args(gpu), runs=c.ints(gpu, c.runs)))
