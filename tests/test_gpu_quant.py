"""The 8-bit cache and the windowed read on the GPU against the float64 oracle (oracle/quant.py).

Codes, scale bytes and values read back are exact. Attention, per output element, with A = sum_j w_j |v_j| from the
oracle (what a relative error of every weight and of their sum moves an output by) and S the largest |score| (log2):
  one query, fp32 out: a weight is a bf16 pair (2^-8 * 2^-8 = 2^-16 relative); its exponent is a product of fp32 sums
      over 128 exact products, at most (S + 8) 2^-20 relative to the weight (7 additions deep in the matrix core and 4
      between them, one multiply, one subtraction: 16 roundings of at most S 2^-24), exp2 itself 2^-22; sums over up to
      2^17 rows in tiles of 32 by four lanes, merged pairwise: 2^-17. Weight and sum err alike: twice the total.
  a chunk: the weights are rounded to bf16 before the product with V, 2^-8, their sum is not.
  bf16 out: half a step, 2^-8 of the value.
"""
from __future__ import annotations

import math
import threading

import numpy as np
import pytest
import torch

from attention_lab import (QuantCache, dequantize_rows, gather_attention, full_attention, quant_attention,
                           quant_gather_attention, quantize_append, window_attention)
from oracle import quant as oq

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128)
LOG2E = math.log2(math.e)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen(seed)).to(dtype)


def bytes_of(t):
    return t.view(torch.uint8).cpu().numpy().copy()


def random_cache(gpu, seed, B, G, C, block):
    """Random codes (no NaN) over random scales, and the values they stand for."""
    g = gen(seed)
    k, v = (torch.randint(0, 255, (B, G, C, 128), generator=g).to(torch.uint8) for _ in "kv")
    for t in (k, v):     # magnitudes up to 1.875 * 2^3: codes below 0x58 of either sign
        t.copy_((t & 128) | (t & 127) % 0x58)
    ke, ve = (torch.randint(121, 126, (B, G, -(-C // block)), generator=g).to(torch.uint8) for _ in "kv")
    cache = QuantCache(k.to(gpu).view(torch.float8_e4m3fn), v.to(gpu).view(torch.float8_e4m3fn), ke.to(gpu), ve.to(gpu),
                       block=block)
    return cache, oq.values(k.numpy(), ke.numpy(), block), oq.values(v.numpy(), ve.numpy(), block)


def f64(t):
    return t.detach().double().cpu().numpy()


def weights_times(fn, v):
    return fn(np.abs(v))


def check(got, want, A, S, *, chunk, what):
    w = (2.0 ** -8 if chunk else 2.0 ** -16) + (S + 8) * 2.0 ** -20 + 2.0 ** -22 + 2.0 ** -17
    tol = 2 * w * A + (2.0 ** -8 * np.abs(want) if got.dtype == torch.bfloat16 else 0) + 1e-30
    g = f64(got)
    np.testing.assert_array_equal(np.isnan(g), np.isnan(want), err_msg=what)
    err = np.where(np.isnan(want), 0, np.abs(g - want))
    bad = err > np.where(np.isnan(tol), np.inf, tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outputs off, worst {np.nanmax(err / tol):.2f} of the bound"


def top_score(q, k):
    """The largest |score| in the log2 domain."""
    kk = np.nan_to_num(np.abs(k), nan=0, posinf=0).max(axis=(0, 1, 2))
    return float((np.abs(q) * kk).sum(-1).max() * SCALE * LOG2E)


# ---------------------------------------------------------------------------------------------------------------------
# writing and reading back
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,G,C,T,start,block,dtype", [
    (1, 1, 64, 1, 0, 64, torch.bfloat16), (2, 3, 200, 1, 37, 16, torch.bfloat16), (1, 2, 200, 1, 199, 32, torch.float32),
    (2, 2, 300, 64, 64, 64, torch.bfloat16), (1, 2, 300, 65, 63, 64, torch.float16), (2, 1, 333, 333, 0, 32, torch.float32),
    (1, 2, 333, 130, 95, 16, torch.bfloat16), (1, 1, 1, 1, 0, 16, torch.float16), (3, 2, 1000, 517, 483, 64, torch.bfloat16)])
def test_append_writes_the_oracles_codes(gpu, B, G, C, T, start, block, dtype):
    cache, _, _ = random_cache(gpu, 1, B, G, C, block)
    want = [(bytes_of(cache.k), bytes_of(cache.k_exp)), (bytes_of(cache.v), bytes_of(cache.v_exp))]
    loud = torch.exp2(torch.randn(B, G, T, 1, generator=gen(3)) * 2)      # rows of different loudness: scales grow
    k = (randn(4, B, G, T, 128, dtype=torch.float32) * loud).to(dtype)
    v = (randn(5, B, G, T, 128, dtype=torch.float32) * 2.0 ** -9).to(dtype)
    quantize_append(cache, k.to(gpu), v.to(gpu), start)
    for (codes, exps), x, c, e in zip(want, (k, v), (cache.k, cache.v), (cache.k_exp, cache.v_exp)):
        oq.append(codes, exps, f64(x), start, block)
        np.testing.assert_array_equal(bytes_of(e), exps)
        np.testing.assert_array_equal(bytes_of(c), codes)     # the new rows, the moved ones and all the others


def test_append_in_steps_grows_scales_and_moves_old_rows(gpu):
    B, G, C, block = 2, 2, 100, 32
    cache = QuantCache.empty(B, G, C, block=block, device=gpu)
    codes, exps = bytes_of(cache.k), bytes_of(cache.k_exp)
    at = 0
    for n, T in enumerate((1, 1, 5, 20, 1, 40, 1, 31)):
        x = (randn(n, B, G, T, 128, dtype=torch.float32) * 2.0 ** (n % 3 * 5 - 4)).to(torch.bfloat16)
        quantize_append(cache, x.to(gpu), x.to(gpu), at)
        oq.append(codes, exps, f64(x), at, block)
        at += T
    assert at == C
    for c, e in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)):
        np.testing.assert_array_equal(bytes_of(e), exps)
        np.testing.assert_array_equal(bytes_of(c), codes)


def test_append_extremes(gpu):
    """Zeros, subnormals, the largest values, NaN and infinities; moves over more than fp32's exponent range."""
    rows = torch.zeros(1, 1, 16, 128)
    rows[0, 0, 1] = 1e-40
    rows[0, 0, 2] = 2.0 ** -119
    rows[0, 0, 3, ::2] = -3e38
    rows[0, 0, 4] = 3.4e38
    rows[0, 0, 5, 7], rows[0, 0, 5, 8], rows[0, 0, 5, 9] = math.nan, math.inf, -math.inf
    rows[0, 0, 6] = 448.0
    rows[0, 0, 7] = 464.0          # rounds to 448 under a scale of 1
    for pick in ([0], [0, 1], [1, 2], [2, 4], [5], [5, 6], [6, 5, 7], list(range(16)), [4, 3, 2, 1]):
        x = rows[:, :, pick]
        cache, _, _ = random_cache(gpu, 7, 1, 1, 40, 16)
        codes, exps = bytes_of(cache.k), bytes_of(cache.k_exp)
        for i in range(len(pick)):
            quantize_append(cache, x[:, :, i:i + 1].to(gpu), x[:, :, i:i + 1].to(gpu), 5 + i)
            oq.append(codes, exps, f64(x[:, :, i:i + 1]), 5 + i, 16)
        got = bytes_of(cache.k)
        np.testing.assert_array_equal(bytes_of(cache.k_exp), exps, err_msg=str(pick))
        nan = (codes & 127) == 127         # a NaN's sign is not defined
        np.testing.assert_array_equal(got[~nan], codes[~nan], err_msg=str(pick))
        assert ((got[nan] & 127) == 127).all()
        assert np.isfinite(f64(dequantize_rows(cache, 0, 40)[0])[~nan]).all()


def test_append_ragged_starts_inside_and_outside(gpu):
    B, G, C, T, block = 6, 2, 150, 70, 32
    starts = [0, 33, 149, -20, 200, 96]
    cache, _, _ = random_cache(gpu, 11, B, G, C, block)
    x = randn(12, B, G, T, 128)
    codes, exps = bytes_of(cache.k), bytes_of(cache.k_exp)
    st = torch.tensor(starts, dtype=torch.int32, device=gpu)
    quantize_append(cache, x.to(gpu), x.to(gpu), st)
    for b, s in enumerate(starts):       # the oracle on the rows that lie inside
        lo, hi = max(s, 0), min(s + T, C)
        if lo < hi:
            oq.append(codes[b:b + 1], exps[b:b + 1], f64(x)[b:b + 1, :, lo - s:hi - s], lo, block)
    np.testing.assert_array_equal(bytes_of(cache.k_exp), exps)
    np.testing.assert_array_equal(bytes_of(cache.k), codes)
    k, _ = dequantize_rows(cache, st, T, dtype=torch.float32)
    want = oq.values(codes, exps, block)
    for b, s in enumerate(starts):
        pos = np.arange(s, s + T)
        ok = (pos >= 0) & (pos < C)
        np.testing.assert_array_equal(f64(k)[b][:, ok], want[b][:, pos[ok]])
        assert (f64(k)[b][:, ~ok] == 0).all()


def test_append_extreme_device_starts(gpu):
    cache, _, _ = random_cache(gpu, 13, 4, 1, 64, 16)
    before = bytes_of(cache.k)
    st = torch.tensor([2 ** 31 - 1, -2 ** 31, 64, -1], dtype=torch.int32, device=gpu)
    x = randn(1, 4, 1, 1, 128).to(gpu)
    quantize_append(cache, x, x, st)
    assert np.array_equal(bytes_of(cache.k), before)
    assert (f64(dequantize_rows(cache, st, 1)[0]) == 0).all()


def test_a_first_write_inside_a_block_takes_its_own_scale(gpu):
    """A sequence that begins inside a block of an empty cache: small rows keep their precision."""
    cache = QuantCache.empty(1, 1, 64, block=64, device=gpu)
    x = randn(3, 1, 1, 20, 128) * 2.0 ** -12
    quantize_append(cache, x.to(gpu), x.to(gpu), 7)
    for t in dequantize_rows(cache, 7, 20, dtype=torch.float32):
        top = float(x.abs().max())
        err = (t.cpu().double() - x.double()).abs()
        assert bool((err <= 2.0 ** -4 * x.double().abs() + 2.0 ** -17 * top).all())


def test_append_takes_any_strides(gpu):
    B, G, T, block = 2, 4, 50, 16
    base = randn(3, B, T, G, 128)
    want, _, _ = random_cache(gpu, 1, B, G, 64, block)
    quantize_append(want, base.transpose(1, 2).contiguous().to(gpu), base.transpose(1, 2).contiguous().to(gpu), 3)
    wide = randn(9, B, T, G, 256).to(gpu)
    wide[..., 64:192] = base.to(gpu)
    odd = torch.zeros(base.numel() + 3, dtype=torch.bfloat16, device=gpu)[3:].view(base.shape).copy_(base.to(gpu))
    last = base.to(gpu).transpose(1, 2).transpose(2, 3).contiguous().transpose(2, 3)
    for x in (base.to(gpu).transpose(1, 2), wide[..., 64:192].transpose(1, 2), odd.transpose(1, 2), last):
        got, _, _ = random_cache(gpu, 1, B, G, 64, block)
        quantize_append(got, x, x, 3)
        assert np.array_equal(bytes_of(got.k), bytes_of(want.k)) and np.array_equal(bytes_of(got.v), bytes_of(want.v))
    one = base[:, :1].to(gpu).transpose(1, 2)
    a, _, _ = random_cache(gpu, 1, B, G, 64, block)
    b, _, _ = random_cache(gpu, 1, B, G, 64, block)
    quantize_append(a, one.expand(B, G, 30, 128), one.expand(B, G, 30, 128), 3)      # stride 0 along T
    quantize_append(b, one.repeat(1, 1, 30, 1), one.repeat(1, 1, 30, 1), 3)
    assert np.array_equal(bytes_of(a.k), bytes_of(b.k))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_read_back_every_code(gpu, dtype):
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 2, 128).repeat(1, 1, 24, 1).contiguous()
    exps = torch.tensor([17, 120, 134], dtype=torch.uint8).view(1, 1, 3)
    cache = QuantCache(codes.to(gpu).view(torch.float8_e4m3fn), codes.to(gpu).view(torch.float8_e4m3fn), exps.to(gpu),
                       exps.to(gpu), block=16)
    want = torch.from_numpy(oq.values(codes.numpy(), exps.numpy(), 16))
    for start, length in ((0, 48), (5, 40), (47, 1), (9, 0)):
        k, v = dequantize_rows(cache, start, length, dtype=dtype)
        w = want[:, :, start:start + length].to(dtype)
        assert k.dtype == dtype and k.shape == w.shape
        assert torch.equal(torch.nan_to_num(k.cpu(), nan=-1.0), torch.nan_to_num(w, nan=-1.0))
        assert torch.equal(torch.nan_to_num(v.cpu(), nan=-1.0), torch.nan_to_num(w, nan=-1.0))


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def a_cache(gpu, kind, seed, B, G, C):
    """(call, k values, v values): the read over a cache of the kind, "bf16" or the 8-bit block size."""
    if kind == "bf16":
        k, v = randn(seed, B, G, C, 128), randn(seed + 1, B, G, C, 128)
        kd, vd = k.to(gpu), v.to(gpu)
        return (lambda q, **kw: window_attention(q, kd, vd, **{"window": None, **kw})), f64(k), f64(v), (kd, vd)
    cache, k, v = random_cache(gpu, seed, B, G, C, kind)
    return (lambda q, **kw: quant_attention(q, cache, **kw)), k, v, (cache.k, cache.v)


def expect(q, k, v, legal, p0, window, sinks, scale=SCALE):
    one = lambda x: oq.range_attention(f64(q), k, x, legal, p0, window, sinks, scale)  # noqa: E731
    return one(v), one(np.abs(v))


@pytest.mark.parametrize("kind", ["bf16", 16, 32, 64])
@pytest.mark.parametrize("h", [1, 2, 3, 8])
@pytest.mark.parametrize("L,window,sinks", [(1, None, 0), (2, 1, 0), (31, None, 0), (32, 5, 4), (33, 33, 4), (129, 64, 0),
                                            (300, None, 0), (300, 37, 5), (300, 100, 250), (299, 1, 1), (160, 1000, 64)])
def test_one_query(gpu, kind, h, L, window, sinks):
    B, G, C = 2, 2, 300
    call, k, v, _ = a_cache(gpu, kind, 5, B, G, C)
    q = randn(17, B, G, h, 1, 128)
    want, A = expect(q, k, v, L, L - 1, window, sinks)
    S = top_score(f64(q), k)
    for P in (None, 1, 3):
        for dt in (torch.float32, torch.bfloat16):
            got = call(q.to(gpu), valid_length=L, window=window, sinks=sinks, partitions=P, out_dtype=dt)
            check(got, want, A, S, chunk=False, what=f"P={P} {dt}")


@pytest.mark.parametrize("kind", ["bf16", 32])
def test_one_query_long_rows_and_many_partitions(gpu, kind):
    B, G, C, h = 1, 2, 9001, 4
    call, k, v, _ = a_cache(gpu, kind, 5, B, G, C)
    q = randn(17, B, G, h, 1, 128)
    S = top_score(f64(q), k)
    for L, window, sinks in ((9001, None, 0), (8888, 4100, 7)):
        want, A = expect(q, k, v, L, L - 1, window, sinks)
        for P in (None, 1, 2, 7, 64, 256):
            got = call(q.to(gpu), valid_length=L, window=window, sinks=sinks, partitions=P, out_dtype=torch.float32)
            check(got, want, A, S, chunk=False, what=f"L={L} P={P}")


@pytest.mark.parametrize("kind", ["bf16", 16, 64])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3), (1, 0)])
def test_one_query_with_a_length_per_sequence(gpu, kind, window, sinks):
    B, G, C, h = 7, 2, 200, 4
    lengths = [0, 1, 200, 64, -3, 999, 131]
    call, k, v, _ = a_cache(gpu, kind, 5, B, G, C)
    q = randn(17, B, G, h, 1, 128)
    n = np.clip(lengths, 0, C)
    want, A = expect(q, k, v, n, n - 1, window, sinks)
    lt = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    for P in (None, 1, 5):
        got = call(q.to(gpu), valid_length=lt, window=window, sinks=sinks, partitions=P, out_dtype=torch.float32)
        check(got, want, A, top_score(f64(q), k), chunk=False, what=f"P={P}")
        assert (f64(got)[[0, 4]] == 0).all()


@pytest.mark.parametrize("kind", ["bf16", 32])
@pytest.mark.parametrize("legal,p,window,sinks", [(100, 40, None, 0), (100, 40, 7, 2), (100, 140, 20, 0), (100, 140, 50, 3),
                                                  (100, 99, 2 ** 31, 2 ** 31), (100, 2 ** 31 - 3, 5, 3)])
def test_one_query_away_from_the_end(gpu, kind, legal, p, window, sinks):
    call, k, v, _ = a_cache(gpu, kind, 5, 1, 2, 130)
    q = randn(17, 1, 2, 2, 1, 128)
    want, A = expect(q, k, v, legal, p, window, sinks)
    for heads in (2, 9):     # nine heads take the chunk kernel
        qq = q[:, :, :1].repeat(1, 1, heads, 1, 1) if heads == 9 else q
        w, a = (want, A) if heads == 2 else (want[:, :, :1].repeat(9, 2), A[:, :, :1].repeat(9, 2))
        got = call(qq.to(gpu), valid_length=legal, query_start=p, window=window, sinks=sinks)
        check(got, w, a, top_score(f64(q), k), chunk=heads == 9, what=f"h={heads}")


@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("S", [1, 31, 33, 200, 5000])
def test_listed_rows(gpu, block, S):
    B, G, C, h = 2, 2, 300, 4
    cache, k, v = random_cache(gpu, 5, B, G, C, block)
    q = randn(17, B, G, h, 1, 128)
    rows = torch.randint(0, C, (B, G, S), generator=gen(S))        # unsorted, and the same row more than once
    rows[:, :, ::7] = torch.tensor([-1, C, -2 ** 31, 2 ** 31 - 1]).repeat(S)[:rows[:, :, ::7].shape[2]]
    rows[0, 1] = -1                                                 # a query with no row
    qf = f64(q)[:, :, :, 0]
    want = oq.listed_attention(qf, k, v, rows.numpy(), SCALE)[:, :, :, None]
    A = oq.listed_attention(qf, k, np.abs(v), rows.numpy(), SCALE)[:, :, :, None]
    for P in (None, 1, 4):
        for r in (rows.to(torch.int32), rows):
            got = quant_gather_attention(q.to(gpu), cache, r.to(gpu), partitions=P, out_dtype=torch.float32)
            check(got, want, A, top_score(f64(q), k), chunk=False, what=f"P={P}")
    far = rows.clone()
    far[rows < 0] = 2 ** 32 + 5          # not position 5
    valid = torch.rand(rows.shape, generator=gen(1)) < 0.5
    got = quant_gather_attention(q.to(gpu), cache, far.to(gpu), valid.to(gpu), out_dtype=torch.float32)
    masked = np.where(valid.numpy(), rows.numpy(), -1)
    check(got, oq.listed_attention(qf, k, v, masked, SCALE)[:, :, :, None],
          oq.listed_attention(qf, k, np.abs(v), masked, SCALE)[:, :, :, None], top_score(f64(q), k), chunk=False,
          what="selected_valid")


def test_listed_rows_equal_the_bfloat16_read_of_the_values(gpu):
    """Beside gather_attention over the dequantised cache: the same values, so the same output up to its rounding."""
    B, G, C, h, S = 2, 4, 4096, 2, 333
    cache, k, v = random_cache(gpu, 5, B, G, C, 64)
    kb, vb = dequantize_rows(cache)
    rows = torch.stack([torch.randperm(C, generator=gen(i))[:S] for i in range(B * G)]).view(B, G, S).to(gpu)
    q = randn(17, B, G, h, 1, 128).to(gpu)
    a, b = quant_gather_attention(q, cache, rows), gather_attention(q, kb, vb, rows)
    err = (a.double() - b.double()).abs()
    assert bool((err <= 2.0 ** -7 * b.double().abs() + 1e-4).all())
    a, b = quant_attention(q, cache, valid_length=4000), full_attention(q, kb, vb, valid_length=4000)
    err = (a.double() - b.double()).abs()
    assert bool((err <= 2.0 ** -7 * b.double().abs() + 1e-4).all())


@pytest.mark.parametrize("kind", ["bf16", 16, 64])
@pytest.mark.parametrize("h,T,past,window,sinks", [
    (1, 2, 0, None, 0), (2, 70, 0, None, 0), (2, 65, 100, None, 0), (4, 33, 200, 40, 5), (3, 90, 31, 17, 0),
    (5, 26, 150, 64, 70), (8, 17, 0, 1, 0), (16, 9, 300, 100, 1), (7, 130, 3, 1000, 4), (1, 129, 128, 64, 64),
    (2, 200, 0, 3, 2), (16, 1, 64, None, 0)])
def test_chunk(gpu, kind, h, T, past, window, sinks):
    B, G = 2, 2
    L = past + T
    C = L + 9
    call, k, v, _ = a_cache(gpu, kind, 5, B, G, C)
    q = randn(17, B, G, h, T, 128)
    want, A = expect(q, k, v, L, past, window, sinks)
    for P in (None, 1, 3, 16):
        got = call(q.to(gpu), valid_length=L, window=window, sinks=sinks, partitions=P)
        check(got, want, A, top_score(f64(q), k), chunk=True, what=f"P={P}")


@pytest.mark.parametrize("kind", ["bf16", 32])
@pytest.mark.parametrize("legal,start,window,sinks", [(50, 20, None, 0), (50, 20, 6, 0), (50, 45, 10, 2), (50, 60, 4, 0),
                                                      (50, 60, 4, 3), (3, 0, None, 0)])
def test_chunk_with_queries_past_the_valid_keys(gpu, kind, legal, start, window, sinks):
    """Queries behind the last valid key, some of which read nothing: zeros."""
    B, G, h, T, C = 1, 2, 2, 40, 120
    call, k, v, _ = a_cache(gpu, kind, 5, B, G, C)
    q = randn(17, B, G, h, T, 128)
    want, A = expect(q, k, v, legal, start, window, sinks)
    for P in (None, 3):
        got = call(q.to(gpu), valid_length=legal, query_start=start, window=window, sinks=sinks, partitions=P)
        check(got, want, A, top_score(f64(q), k), chunk=True, what=f"P={P}")


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-30])
@pytest.mark.parametrize("kind", ["bf16", 16])
def test_scales(gpu, kind, scale):
    call, k, v, _ = a_cache(gpu, kind, 5, 1, 2, 100)
    for T in (1, 30):
        q = randn(17, 1, 2, 2, T, 128)
        want, A = expect(q, k, v, 90, 90 - T, 50, 3, scale)
        got = call(q.to(gpu), valid_length=90, window=50, sinks=3, scale=scale)
        check(got, want, A, top_score(f64(q), k) / SCALE * abs(scale), chunk=T > 1, what=f"T={T}")


@pytest.mark.parametrize("kind,poison", [("bf16", math.nan), ("bf16", math.inf), ("bf16", -math.inf), (16, math.nan),
                                         (64, math.nan)])
def test_masked_places_never_matter(gpu, kind, poison):
    """Whatever lies past the valid length, between the sinks and the window, or ahead of a query stays out of its
    output: NaN codes in the 8-bit cache (e4m3 has no infinity), NaN and infinities in the bfloat16 one."""
    B, G, h, C = 1, 2, 2, 260
    call, k, v, (kt, vt) = a_cache(gpu, kind, 5, B, G, C)
    q1 = randn(17, B, G, h, 1, 128)

    def spoil(lo, hi):
        for t, x in ((kt, k), (vt, v)):
            if kind == "bf16":
                t[:, :, lo:hi] = poison
            else:
                t.view(torch.uint8)[:, :, lo:hi] = 0x7f
            x[:, :, lo:hi] = poison

    keep = [(kt.clone(), k.copy()), (vt.clone(), v.copy())]

    def restore():
        for (t, x), a, b in zip(keep, (kt, vt), (k, v)):
            a.copy_(t)
            b[:] = x

    spoil(200, C)
    spoil(5, 150)
    want, A = expect(q1, k, v, 200, 199, 50, 5)
    assert np.isfinite(want).all()
    for P in (1, 4):
        check(call(q1.to(gpu), valid_length=200, window=50, sinks=5, partitions=P), want, A, top_score(f64(q1), k),
              chunk=False, what="one query")
    restore()
    # a chunk of 60 at 140: position 170 is spoilt, which the first 30 queries do not see and the others do (NaN); and
    # positions 8..99, which the window of the last 20 excludes and that of the first ones includes
    spoil(170, 171)
    spoil(200, C)
    q = randn(19, B, G, h, 60, 128)
    for lo, hi, window, sinks in ((0, 0, None, 0), (8, 100, 60, 8)):
        spoil(lo, hi)
        with np.errstate(invalid="ignore"):
            want, A = expect(q, k, v, 200, 140, window, sinks)
        assert np.isfinite(want[:, :, :, 22:30]).all()
        for P in (1, 3):
            got = call(q.to(gpu), valid_length=200, query_start=140, window=window, sinks=sinks, partitions=P)
            fin = np.isfinite(want)
            g = f64(got)
            # a query that sees a spoilt row has no finite value of its own; the others keep theirs
            seen = ~fin.all(axis=-1, keepdims=True) & np.ones_like(fin)
            assert not np.isfinite(g[~fin]).any()
            check(torch.from_numpy(np.where(seen, 0, g)).to(torch.bfloat16), np.where(seen, 0, want),
                  np.where(seen, 0, np.nan_to_num(A)), top_score(f64(q), k), chunk=True, what=f"chunk P={P}")
    restore()


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16])
def test_listed_rows_of_narrow_types(gpu, dtype):
    """A skipped slot is no position in any type: 255 is what -1 would be in uint8."""
    B, G, C, h, S = 1, 2, 300, 2, 40
    cache, k, v = random_cache(gpu, 6, B, G, C, 32)
    q = randn(18, B, G, h, 1, 128)
    rows = torch.randint(0, 100, (B, G, S), generator=gen(S))
    valid = torch.rand(rows.shape, generator=gen(2)) < 0.5
    valid[0, 1] = False
    masked = np.where(valid.numpy(), rows.numpy(), -1)
    qf = f64(q)[:, :, :, 0]
    got = quant_gather_attention(q.to(gpu), cache, rows.to(dtype).to(gpu), valid.to(gpu), out_dtype=torch.float32)
    check(got, oq.listed_attention(qf, k, v, masked, SCALE)[:, :, :, None],
          oq.listed_attention(qf, k, np.abs(v), masked, SCALE)[:, :, :, None], top_score(f64(q), k), chunk=False,
          what=str(dtype))


@pytest.mark.parametrize("dtype", [torch.bool, torch.float32, torch.complex64, torch.uint16, torch.uint32, torch.uint64])
def test_listed_rows_of_other_types_are_refused(gpu, dtype):
    cache, _, _ = random_cache(gpu, 6, 1, 2, 64, 32)
    q = randn(18, 1, 2, 2, 1, 128).to(gpu)
    with pytest.raises(ValueError, match="integer"):
        quant_gather_attention(q, cache, torch.zeros(1, 2, 8, dtype=dtype, device=gpu))


@pytest.mark.parametrize("kind", ["bf16", 16])
@pytest.mark.parametrize("B,G,C,h,partitions", [(130, 1, 200, 1, None), (130, 1, 200, 1, 256), (65, 2, 90, 3, 2),
                                                (5, 1, 3000, 2, 256)])
def test_a_length_for_each_of_many_sequences(gpu, kind, B, G, C, h, partitions):
    """More sequences than a wave has lanes, more partitions than tiles, empty sequences among them."""
    call, k, v, _ = a_cache(gpu, kind, 12, B, G, C)
    q = randn(19, B, G, h, 1, 128)
    lengths = torch.randint(0, C + 1, (B,), generator=gen(B))
    lengths[::9] = 0
    lengths[1], lengths[-1] = C, 1
    got = call(q.to(gpu), valid_length=lengths.to(torch.int32).to(gpu), window=None, sinks=0, out_dtype=torch.float32,
               partitions=partitions)
    S = top_score(f64(q), k)
    for b in range(B):
        if lengths[b] == 0:
            assert not got[b].any()
            continue
        w, a = expect(q[b:b + 1], k[b:b + 1], v[b:b + 1], int(lengths[b]), int(lengths[b]) - 1, None, 0)
        check(got[b:b + 1], w, a, S, chunk=False, what=f"b={b}")


@pytest.mark.parametrize("kind", ["bf16", 64])
@pytest.mark.parametrize("B,C,h,partitions", [(1, 2112, 2, None), (4, 2112, 8, 16), (32, 700, 3, 4), (2, 9000, 1, 8)])
def test_a_length_each_in_one_launch_and_in_two(gpu, kind, B, C, h, partitions):
    """Small ragged calls merge in their launch and captured ones in a second: the same bits, whatever the lengths, call
    after call (the counters return to zero)."""
    G = 2
    call, k, v, _ = a_cache(gpu, kind, 22, B, G, C)
    q = randn(23, B, G, h, 1, 128).to(gpu)
    lengths = torch.zeros(B, dtype=torch.int32, device=gpu)
    read = lambda: call(q, valid_length=lengths, window=None, sinks=0, out_dtype=torch.float32,  # noqa: E731
                        partitions=partitions)
    read()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = read()
    S = top_score(f64(q), k)
    for fill in ([C] * B, [0] * B, [1] * B, [C if b == B // 2 else 40 for b in range(B)],
                 torch.randint(0, C + 1, (B,), generator=gen(B)).tolist()):
        lengths.copy_(torch.tensor(fill, dtype=torch.int32))
        eager = read()
        graph.replay()
        assert torch.equal(eager, out)
        b = B // 2
        if fill[b] == 0:
            assert not eager.any()
        else:
            w, a = expect(q[b:b + 1], k[b:b + 1], v[b:b + 1], fill[b], fill[b] - 1, None, 0)
            check(eager[b:b + 1], w, a, S, chunk=False, what=str(fill[b]))


@pytest.mark.parametrize("B,G,C,h,partitions", [(4200, 1, 40, 1, 2), (40, 2, 600, 8, 16), (8, 4, 600, 8, 16)])
def test_more_rows_than_the_shared_partials_hold(gpu, B, G, C, h, partitions):
    """Past the counters, past the partials, and at the partials' last row; repeated, so the counters are zero again."""
    call, k, v, _ = a_cache(gpu, 32, 13, B, G, C)
    q = randn(20, B, G, h, 1, 128)
    first = call(q.to(gpu), window=None, sinks=0, out_dtype=torch.float32, partitions=partitions)
    w, a = expect(q, k, v, C, C - 1, None, 0)
    check(first, w, a, top_score(f64(q), k), chunk=False, what="first")
    for _ in range(3):
        again = call(q.to(gpu), window=None, sinks=0, out_dtype=torch.float32, partitions=partitions)
        assert torch.equal(first, again)


@pytest.mark.parametrize("kind", ["bf16", 16, 64])
@pytest.mark.parametrize("window,sinks", [(None, 0), (200, 0), (65, 70)])
@pytest.mark.parametrize("partitions", [1, 3])
def test_chunk_with_values_that_are_not_numbers(gpu, kind, window, sinks, partitions):
    """NaN rows of V inside the chunk and its history: the queries that see one get NaN, every other one its output."""
    B, G, h, T, past = 1, 2, 2, 300, 700
    C = past + T + 20
    call, k, v, (_, vt) = a_cache(gpu, kind, 14, B, G, C)
    q = randn(21, B, G, h, T, 128)
    spoilt = [past + T - 2, past + T + 3] + ([] if window is None else [past + 3, sinks + 7])
    for p in spoilt:
        v[0, 1, p] = np.nan
        if kind == "bf16":
            vt[0, 1, p] = math.nan
        else:
            vt.view(torch.uint8)[0, 1, p] = 0x7f
    L = past + T
    got = call(q.to(gpu), valid_length=L, query_start=past, window=window, sinks=sinks, partitions=partitions)
    w, _ = expect(q, k, v, L, past, window, sinks)
    _, a = expect(q, k, np.nan_to_num(v), L, past, window, sinks)
    assert np.isnan(w).any() and not np.isnan(w[0, 0]).any() and not np.isnan(w).all(axis=(2, 3, 4)).any()
    check(got, w, a, top_score(f64(q), k), chunk=True, what=f"{kind} {window} {sinks}")


@pytest.mark.parametrize("kind", ["bf16", 16])
def test_large_scores_and_minus_infinity(gpu, kind):
    """Scores hundreds apart; a query whose every score is -inf gets zeros (bfloat16 cache)."""
    B, G, h, C = 1, 1, 2, 96
    call, k, v, (kt, vt) = a_cache(gpu, kind, 5, B, G, C)
    for T in (1, 20):
        q = randn(17, B, G, h, T, 128) * 60
        want, A = expect(q, k, v, 96, 96 - T, None, 0)
        check(call(q.to(gpu), valid_length=96), want, A, top_score(f64(q), k), chunk=T > 1, what=f"T={T}")
        if kind == "bf16":
            spoilt = kt.clone()
            spoilt[..., 0] = -math.inf
            q[..., 0] = 1.0
            got = window_attention(q.to(gpu), spoilt, vt, window=None)
            assert (f64(got) == 0).all()


def test_offsets_past_32_bits(gpu):
    """A cache whose codes and whose bf16 rows lie past 2^32 bytes."""
    B, G, C, h = 1, 2, 9_000_000, 2
    cache = QuantCache.empty(B, G, C, device=gpu)
    x = randn(3, B, G, 100, 128)
    quantize_append(cache, x.to(gpu), x.to(gpu), C - 100)
    kv = dequantize_rows(cache, C - 100, 100)
    assert float((kv[0].float().cpu() - x.float()).abs().max()) <= 2.0 ** -4 * 4.5
    k, v = (f64(t) for t in kv)
    for T in (1, 40):
        q = randn(17, B, G, h, T, 128)
        want = oq.range_attention(f64(q), k, v, 100, 100 - T, 30, 0, SCALE)
        A = oq.range_attention(f64(q), k, np.abs(v), 100, 100 - T, 30, 0, SCALE)
        got = quant_attention(q.to(gpu), cache, valid_length=C, window=30)
        check(got, want, A, top_score(f64(q), k), chunk=T > 1, what=f"T={T}")
    rows = torch.arange(C - 60, C - 20, dtype=torch.int32).view(1, 1, -1).expand(1, 2, -1)
    q = randn(17, B, G, h, 1, 128)
    got = quant_gather_attention(q.to(gpu), cache, rows.to(gpu))
    at = rows.numpy() - (C - 100)
    check(got, oq.listed_attention(f64(q)[:, :, :, 0], k, v, at, SCALE)[:, :, :, None],
          oq.listed_attention(f64(q)[:, :, :, 0], k, np.abs(v), at, SCALE)[:, :, :, None], top_score(f64(q), k), chunk=False,
          what="rows")
    del cache
    big = torch.empty(1, 2, 17_000_000, 128, dtype=torch.bfloat16, device=gpu)
    big[:, :, -100:] = x.to(gpu)
    for T in (1, 40):
        q = randn(17, B, G, h, T, 128)
        want = oq.range_attention(f64(q), f64(x), f64(x), 100, 100 - T, 30, 0, SCALE)
        A = oq.range_attention(f64(q), f64(x), np.abs(f64(x)), 100, 100 - T, 30, 0, SCALE)
        check(window_attention(q.to(gpu), big, big, window=30, sinks=0), want, A, top_score(f64(q), f64(x)), chunk=T > 1,
              what=f"bf16 T={T}")


def test_results_repeat_bit_for_bit(gpu):
    for kind in ("bf16", 32):
        call, _, _, _ = a_cache(gpu, kind, 5, 2, 4, 5000)
        for T in (1, 150):
            q = randn(17, 2, 4, 4, T, 128).to(gpu)
            first = call(q, valid_length=4800, window=3000, sinks=4)
            for _ in range(3):
                assert torch.equal(call(q, valid_length=4800, window=3000, sinks=4), first)


# ---------------------------------------------------------------------------------------------------------------------
# as a program uses them
# ---------------------------------------------------------------------------------------------------------------------
def test_a_prompt_and_tokens_together(gpu):
    """A prompt in two chunks and decode steps: write, causal chunk, window, a list; every output against the oracle on
    the oracle's own cache."""
    B, G, h, C, block = 2, 2, 4, 256, 32
    cache = QuantCache.empty(B, G, C, block=block, device=gpu)
    kc, ke, vc, ve = (bytes_of(t) for t in (cache.k, cache.k_exp, cache.v, cache.v_exp))
    at = 0
    for n, T in enumerate((90, 47, 1, 1, 1, 60, 1)):
        k, v, q = randn(3 * n, B, G, T, 128), randn(3 * n + 1, B, G, T, 128), randn(3 * n + 2, B, G, h, T, 128)
        quantize_append(cache, k.to(gpu), v.to(gpu), at)
        oq.append(kc, ke, f64(k), at, block)
        oq.append(vc, ve, f64(v), at, block)
        at += T
        kk, vv = oq.values(kc, ke, block), oq.values(vc, ve, block)
        kk[:, :, at:], vv[:, :, at:] = 0, 0     # not read
        S = top_score(f64(q), kk)
        for window, sinks in ((None, 0), (40, 4)):
            want, A = expect(q, kk, vv, at, at - T, window, sinks)
            got = quant_attention(q.to(gpu), cache, valid_length=at, window=window, sinks=sinks)
            check(got, want, A, S, chunk=T > 1, what=f"T={T} window={window}")
        if T == 1:
            rows = torch.cat([torch.arange(4), torch.arange(at - 30, at)]).view(1, 1, -1).expand(B, G, -1)
            got = quant_gather_attention(q.to(gpu), cache, rows.to(gpu))
            check(got, *expect(q, kk, vv, at, at - 1, 30, 4), S, chunk=False, what="rows")
    got = dequantize_rows(cache, 0, at, dtype=torch.float32)
    np.testing.assert_array_equal(f64(got[0]), oq.values(kc, ke, block)[:, :, :at])
    np.testing.assert_array_equal(f64(got[1]), oq.values(vc, ve, block)[:, :, :at])


def test_a_captured_step_follows_its_lengths(gpu):
    """Write and read in one graph with starts and lengths on the device: replays at later positions, between eager work
    of other shapes, equal the eager calls on a cache of their own."""
    B, G, h, C = 3, 2, 2, 400
    caches = [random_cache(gpu, 5, B, G, C, 32)[0] for _ in range(2)]
    pos = torch.tensor([100, 37, 250], dtype=torch.int32, device=gpu)
    length = pos + 1
    x, q = randn(1, B, G, 1, 128).to(gpu), randn(2, B, G, h, 1, 128).to(gpu)

    def step(c):
        quantize_append(c, x, x, pos)
        return (quant_attention(q, c, valid_length=length), quant_attention(q, c, valid_length=length, window=50, sinks=4),
                *dequantize_rows(c, pos, 1))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for n in range(4):
        x.copy_(randn(10 + n, B, G, 1, 128).to(gpu) * (1 + n))
        q.copy_(randn(20 + n, B, G, h, 1, 128).to(gpu))
        graph.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        assert torch.equal(caches[0].k.view(torch.uint8), caches[1].k.view(torch.uint8))
        pos += 1
        length += 1
        quant_attention(randn(3, B, G, 8, 77, 128).to(gpu), caches[1], valid_length=300)   # other shapes between


def test_two_graphs_and_two_streams(gpu):
    """Two captured reads and eager ones on two streams at once share nothing."""
    B, G, h, C = 1, 2, 4, 6000
    call, _, _, _ = a_cache(gpu, 32, 5, B, G, C)
    qs = [randn(i, B, G, h, 1, 128).to(gpu) for i in range(2)]
    want = [call(q, valid_length=5900) for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(q, valid_length=5900))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        eager = []
        for s, g, q in zip(streams, graphs, qs):
            with torch.cuda.stream(s):
                g.replay()
                eager.append([call(q, valid_length=5900) for _ in range(3)])
        torch.cuda.synchronize()
        for o, e, w in zip(outs, eager, want):
            assert torch.equal(o, w) and all(torch.equal(x, w) for x in e)


@pytest.mark.parametrize("own_streams", [False, True])
def test_calls_from_two_threads(gpu, own_streams):
    """Two host threads that read at once, each on its own stream or both on one: the results of one after the other."""
    B, G, C, h = 2, 4, 3000, 4
    call, _, _, _ = a_cache(gpu, 32, 24, B, G, C)
    qs = [randn(60 + i, B, G, h, 1, 128).to(gpu) for i in range(8)]
    want = [call(q, window=None, sinks=0, partitions=8) for q in qs]
    torch.cuda.synchronize()
    shared, failed = torch.cuda.Stream(), []

    def reads():
        try:
            with torch.cuda.stream(torch.cuda.Stream() if own_streams else shared):
                for _ in range(25):
                    got = [call(q, window=None, sinks=0, partitions=8) for q in qs]
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(g, w) for g, w in zip(got, want)):
                failed.append("another result")
        except Exception as e:  # noqa: BLE001 - a thread's exception would be lost
            failed.append(e)

    threads = [threading.Thread(target=reads) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_refusals(gpu):
    cache, _, _ = random_cache(gpu, 5, 2, 2, 100, 32)
    q = randn(1, 2, 2, 2, 1, 128).to(gpu)
    x = randn(1, 2, 2, 3, 128).to(gpu)
    ok = torch.zeros(2, dtype=torch.int32, device=gpu)
    for call, match in (
            (lambda: quantize_append(cache, x, x, 98), "outside"),
            (lambda: quantize_append(cache, x, x[:, :, :2], 0), "must be"),
            (lambda: quantize_append(cache, x, x.float(), 0), "both be"),
            (lambda: quantize_append(cache, x.double(), x.double(), 0), "both be"),
            (lambda: quantize_append(cache, x.cpu(), x.cpu(), 0), "device"),
            (lambda: quantize_append(cache, x, x, ok.long()), "int32"),
            (lambda: quantize_append(cache, x, x, ok.cpu()), "int32"),
            (lambda: dequantize_rows(cache, 90, 11), "outside"),
            (lambda: dequantize_rows(cache, ok), "length"),
            (lambda: dequantize_rows(cache, 0, 3, dtype=torch.float64), "dtype"),
            (lambda: dequantize_rows(cache, 0, -1), "negative"),
            (lambda: quant_attention(q.float(), cache), "bfloat16"),
            (lambda: quant_attention(q[:1], cache), "must be"),
            (lambda: quant_attention(q, cache, valid_length=0), "valid_length"),
            (lambda: quant_attention(q, cache, valid_length=101), "valid_length"),
            (lambda: quant_attention(q, cache, window=0), "window"),
            (lambda: quant_attention(q, cache, window=4, sinks=-1), "sinks"),
            (lambda: quant_attention(q, cache, valid_length=ok[:1]), "int32"),
            (lambda: quant_attention(q, cache, valid_length=ok, query_start=3), "length per sequence"),
            (lambda: quant_attention(q.expand(2, 2, 2, 3, 128), cache, valid_length=ok), "length per sequence"),
            (lambda: quant_attention(q[:, :, :1].expand(2, 2, 9, 1, 128), cache, valid_length=ok), "h <= 8"),
            (lambda: quant_attention(q[:, :, :1].expand(2, 2, 17, 1, 128), cache), "h=17"),
            (lambda: quant_attention(q, cache, valid_length=2, query_start=-1), "non-negative"),
            (lambda: quant_attention(q, cache, query_start=2 ** 31), "2\\^31"),
            (lambda: quant_attention(q.expand(2, 2, 2, 3, 128), cache, valid_length=2), "non-negative"),
            (lambda: quant_attention(q.expand(2, 2, 2, 3, 128), cache, out_dtype=torch.float32), "bfloat16"),
            (lambda: quant_attention(q, cache, partitions=300), "partitions"),
            (lambda: quant_attention(q.expand(2, 2, 2, 3, 128), cache, partitions=17), "partitions"),
            (lambda: quant_attention(q, cache, out=q.float()), "out"),
            (lambda: quant_gather_attention(q, cache, torch.zeros(2, 2, 0, device=gpu, dtype=torch.int32)), "at least one"),
            (lambda: quant_gather_attention(q, cache, torch.zeros(2, 2, 3, device=gpu)), "integer"),
            (lambda: quant_gather_attention(q, cache, torch.zeros(2, 2, 3, dtype=torch.int32)), "device"),
            (lambda: window_attention(q, x, x.float(), window=3), "match"),
            (lambda: QuantCache(cache.k, cache.v, cache.k_exp[:, :, :3], cache.v_exp, block=32), "k_exp"),
            (lambda: QuantCache(cache.k, cache.v[:1], cache.k_exp, cache.v_exp, block=32), "match")):
        with pytest.raises(ValueError, match=match):
            call()
    assert quant_attention(q.expand(2, 2, 2, 1, 128)[:, :, :, :0], cache).shape == (2, 2, 2, 0, 128)
