"""Logits with a common part, which changes no probability: the same order and values, and no more time, as the bound of the largest
logits is as near there."""
from __future__ import annotations

import pytest
import torch

from attention_lab import token_logprobs
from test_gpu_logprobs import check, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,V,top", [(3, 151936, 20), (70, 20011, 64), (2, 32003, 5), (5, 2050, 33)])
@pytest.mark.parametrize("shift", [1000.0, -1000.0, 30000.0])
def test_values(gpu, dtype, N, V, top, shift):
    x = (shift + 2.5 * torch.randn(N, V, generator=gen(V))).to(dtype)
    check(x, torch.randint(0, V, (N,), generator=gen(1)), top, gpu=gpu)


def test_crowded_beside_sparse(gpu):
    """Rows whose largest logits share their upper bits with some, none or all of the others."""
    x = torch.randn(6, 40000, generator=gen(2))
    x[1] = 1000 + 0.01 * x[1]
    x[2, 100:160] = 4096 + torch.arange(60) / 64
    x[3] = 1.0 + x[3].abs() * 2.0 ** -20
    x[4] = -1e-30 * x[4].abs()
    x[5, :20000] += 100000
    for top in (1, 8, 9, 20, 64):
        check(x, torch.arange(6), top, gpu=gpu)


def test_time(gpu):
    """64 float32 rows of a vocabulary, top 20: no more than three times as long around 1000 as around 0 (it was eleven)."""
    base = 2.5 * torch.randn(64, 151936, generator=gen(3))

    def us(x):
        took = []
        for _ in range(7):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(20):
                token_logprobs(x, top=20)
            b.record()
            torch.cuda.synchronize()
            took.append(a.elapsed_time(b) * 50)
        return sorted(took)[3]

    near, far = us(base.to(gpu)), us((base + 1000).to(gpu))
    assert far <= 3 * near, (near, far)
