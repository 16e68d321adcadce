"""The 8-bit cache and the windowed read at the edges of what they take: rows and queries at any address, values near the
largest, and scale bytes of blocks that no row read lies in. Tolerances as in test_gpu_quant.py."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from attention_lab import (QuantCache, dequantize_rows, quant_attention, quant_gather_attention, quantize_append,
                           window_attention)
from oracle import quant as oq
from test_gpu_quant import bytes_of, check, f64, random_cache, randn

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


# ---------------------------------------------------------------------------------------------------------------------
# values near the largest: weights are at most 1, so n rows of less than 2^128 / n have finite sums
# ---------------------------------------------------------------------------------------------------------------------
def loud_rows(gpu, kind, C):
    """K rows that score 0 up to 128 and 7.5 (log2) behind, V rows of one sign up to 1.875 * 2^118; the call and both."""
    g = torch.Generator().manual_seed(3)
    k = torch.zeros(1, 2, C, 128)
    k[:, :, 128:, 0] = 7.5
    codes = torch.randint(0x38, 0x40, (1, 2, C, 128), generator=g).to(torch.uint8)      # 1 to 1.875
    v = codes.view(torch.float8_e4m3fn).double() * 2.0 ** 118
    if kind == "bf16":
        kd, vd = k.to(torch.bfloat16).to(gpu), v.to(torch.bfloat16).to(gpu)
        return (lambda q, **kw: window_attention(q, kd, vd, window=None, **kw)), f64(k), f64(v), None
    nb = -(-C // kind)
    cache = QuantCache(k.to(torch.float8_e4m3fn).to(gpu), codes.to(gpu).view(torch.float8_e4m3fn),
                       torch.full((1, 2, nb), 127, dtype=torch.uint8, device=gpu),
                       torch.full((1, 2, nb), 127 + 118, dtype=torch.uint8, device=gpu), block=kind)
    return (lambda q, **kw: quant_attention(q, cache, **kw)), f64(k), f64(v), cache


@pytest.mark.parametrize("kind", ["bf16", 16, 64])
@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("partitions", [1, 2])
def test_loud_values_have_finite_outputs(gpu, kind, T, partitions):
    C = 300
    call, k, v, cache = loud_rows(gpu, kind, C)
    q = torch.zeros(1, 2, 2, T, 128, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    scale = math.log(2.0)
    want = oq.range_attention(f64(q), k, v, C, C - T, None, 0, scale)
    assert np.isfinite(want.astype(np.float32)).all()
    for dt in (torch.bfloat16, torch.float32) if T == 1 else (torch.bfloat16,):
        got = call(q.to(gpu), scale=scale, out_dtype=dt, partitions=partitions)
        check(got, want, want, 7.5, chunk=T > 1, what=f"{kind} {dt}")
    if T == 1 and cache is not None:
        rows = torch.randperm(C, generator=torch.Generator().manual_seed(1))[:250].view(1, 1, -1).expand(1, 2, -1)
        rows = rows.sort(dim=-1).values     # the quiet rows first
        want = oq.listed_attention(f64(q)[:, :, :, 0], k, v, rows.numpy(), scale)[:, :, :, None]
        got = quant_gather_attention(q.to(gpu), cache, rows.to(gpu), scale=scale, partitions=partitions)
        check(got, want, want, 7.5, chunk=False, what="rows")


@pytest.mark.parametrize("T", [1, 5])
def test_one_row_of_the_largest_value(gpu, T):
    """What the append stores at most, 1.875 * 2^127, is read as it is."""
    cache = QuantCache.empty(1, 1, 64, block=16, device=gpu)
    x = torch.full((1, 1, 1, 128), 3.4e38, device=gpu)
    quantize_append(cache, torch.zeros_like(x), x, 0)
    q = randn(1, 1, 1, 2, T, 128).to(gpu)
    got = quant_attention(q, cache, valid_length=1, query_start=0)
    assert (f64(got) == 1.875 * 2.0 ** 127).all()
    if T == 1:
        got = quant_gather_attention(q, cache, torch.zeros(1, 1, 1, dtype=torch.int32, device=gpu), out_dtype=torch.float32)
        assert (f64(got) == 1.875 * 2.0 ** 127).all()


# ---------------------------------------------------------------------------------------------------------------------
# scale bytes of blocks that no row read lies in
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("byte", [0, 255])
@pytest.mark.parametrize("block", [16, 32, 64])
def test_scale_bytes_of_unread_blocks_never_matter(gpu, byte, block):
    """A cache of the caller's own tensors need not have set the scale bytes of blocks that hold no row yet, or that no
    query reads: whatever they are, and whatever the codes there, the outputs are the same."""
    B, G, h, C = 1, 2, 3, 256
    cache, _, _ = random_cache(gpu, 5, B, G, C, block)
    spoilt, _, _ = random_cache(gpu, 5, B, G, C, block)

    def spoil(keep):
        """Every block without a position of `keep`: its scale byte, and zeros and other codes in its rows."""
        used = torch.zeros(C, dtype=torch.bool)
        used[list(keep)] = True
        for j in range(C // block):
            if not used[block * j:block * j + block].any():
                for t in (spoilt.k_exp, spoilt.v_exp):
                    t[:, :, j] = byte
                for t in (spoilt.k, spoilt.v):
                    t.view(torch.uint8)[:, :, block * j:block * j + block:2] = 0

    q = randn(17, B, G, h, 1, 128).to(gpu)
    rows = torch.tensor([-1, 130, 200, C, 131, -7, 255, 130] * 9, dtype=torch.int32, device=gpu).expand(B, G, -1)
    spoil((130, 131, 200, 255))
    for P in (1, 2):
        assert torch.equal(quant_gather_attention(q, spoilt, rows, partitions=P),
                           quant_gather_attention(q, cache, rows, partitions=P))
    for L, window, sinks in ((130, None, 0), (131, 20, 3), (200, 17, 0)):
        for T in (1, 9):
            keep = set(range(sinks)) | set(range(max(0, L - T - window + 1) if window else 0, L))
            spoilt, _, _ = random_cache(gpu, 5, B, G, C, block)
            spoil(keep)
            qq = randn(18, B, G, h, T, 128).to(gpu)
            for P in (1, 2):
                read = lambda c: quant_attention(qq, c, valid_length=L, window=window, sinks=sinks, partitions=P)  # noqa: E731, B023
                assert torch.equal(read(spoilt), read(cache)), (L, window, sinks, T, P)

