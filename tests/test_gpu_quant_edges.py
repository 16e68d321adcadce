"""The 8-bit cache and the windowed read at the edges of what they take: rows and queries at any address."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from attention_lab import dequantize_rows, quant_attention, quant_gather_attention, quantize_append, window_attention
from test_gpu_quant import bytes_of, random_cache, randn

pytestmark = pytest.mark.gpu


def at_offset(t, elements):
    """t's values, contiguous, `elements` behind an aligned address."""
    return torch.zeros(t.numel() + elements, dtype=t.dtype, device=t.device)[elements:].view(t.shape).copy_(t)


# ---------------------------------------------------------------------------------------------------------------------
# addresses and strides
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("elements", [1, 3])
def test_append_takes_contiguous_rows_at_any_address(gpu, dtype, elements):
    B, G, T, block = 2, 2, 9, 16
    x = randn(3, B, G, T, 128, dtype=dtype).to(gpu)
    odd = at_offset(x, elements)
    assert odd.is_contiguous() and odd.data_ptr() % 16
    want, got = random_cache(gpu, 1, B, G, 64, block)[0], random_cache(gpu, 1, B, G, 64, block)[0]
    quantize_append(want, x, x, 3)
    quantize_append(got, odd, odd, 3)
    for name in ("k", "v", "k_exp", "v_exp"):
        assert np.array_equal(bytes_of(getattr(got, name)), bytes_of(getattr(want, name))), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,G,T", [(1, 1, 1), (1, 2, 1), (2, 1, 1), (1, 1, 5)])
def test_append_takes_any_stride_of_a_dimension_of_one(gpu, dtype, B, G, T):
    """A dimension of one position has no stride that matters, whatever torch keeps there."""
    x = randn(4, B, G, T, 128, dtype=dtype).to(gpu)
    strides = [131 if n == 1 else s for n, s in zip((B, G, T), x.stride())] + [1]
    odd = torch.as_strided(x, x.shape, strides)
    assert torch.equal(odd, x)
    want, got = random_cache(gpu, 1, B, G, 64, 32)[0], random_cache(gpu, 1, B, G, 64, 32)[0]
    quantize_append(want, x, x, 30)
    quantize_append(got, odd, odd, 30)
    for name in ("k", "v", "k_exp", "v_exp"):
        assert np.array_equal(bytes_of(getattr(got, name)), bytes_of(getattr(want, name))), name


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("elements", [1, 4])
def test_reads_take_a_query_at_any_address(gpu, T, elements):
    B, G, h, C = 1, 2, 4, 300
    cache, _, _ = random_cache(gpu, 5, B, G, C, 32)
    kb, vb = dequantize_rows(cache)
    q = randn(17, B, G, h, T, 128).to(gpu)
    odd = at_offset(q, elements)
    assert odd.is_contiguous() and odd.data_ptr() % 16
    assert torch.equal(quant_attention(odd, cache, valid_length=290), quant_attention(q, cache, valid_length=290))
    read = lambda x: window_attention(x, kb, vb, window=70, valid_length=290)  # noqa: E731
    assert torch.equal(read(odd), read(q))
    if T == 1:
        rows = torch.arange(0, 290, 7, dtype=torch.int32, device=gpu).expand(B, G, -1)
        assert torch.equal(quant_gather_attention(odd, cache, rows), quant_gather_attention(q, cache, rows))


@pytest.mark.parametrize("dtype,elements", [(torch.bfloat16, 1), (torch.float32, 1)])
def test_an_output_whose_rows_are_not_aligned_is_refused(gpu, dtype, elements):
    cache, _, _ = random_cache(gpu, 5, 1, 2, 100, 32)
    q = randn(17, 1, 2, 2, 1, 128).to(gpu)
    out = at_offset(torch.zeros(q.shape, dtype=dtype, device=gpu), elements)
    with pytest.raises(ValueError, match="aligned"):
        quant_attention(q, cache, out=out, out_dtype=dtype)
    assert not out.any()
