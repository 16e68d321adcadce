"""The 8-bit K/V cache: rows quantised as they are written, read back, and attended over in place.

A `QuantCache` holds one layer's K and V as e4m3 codes [B,G,C,128] and one scale byte x per block of 16, 32 or 64
positions, KV head and tensor; a value is code * 2^(x - 127), exact in bfloat16. Half the bytes of the bfloat16 cache,
and about half the time of a read of every position (16 requests of 32K, 8 groups, h=4: 161 us for 329), for a rounding of
at most 2^-4 of each value (e4m3 keeps 4 significant bits; values below 2^-14 of their block's largest keep fewer). The sparse
step gains no time by it: its read is of few rows, bound by latencies, and a launch of its own here (80 us a layer for 72).

    cache = QuantCache.empty(B, G, C, device=dev)
    quantize_append(cache, k_prompt, v_prompt, 0)                       # rows [0, T)
    out = quant_attention(q_prompt, cache, valid_length=T)              # the causal chunk
    quantize_append(cache, k_new, v_new, T)                             # one token
    out = quant_attention(q_new, cache, valid_length=T + 1)             # one query, every legal position
    out = quant_attention(q_new, cache, valid_length=T + 1, window=4096, sinks=4)
    out = quant_gather_attention(q_new, cache, rows)                    # one query, the rows of a selection
    k, v = dequantize_rows(cache, 0, T + 1)

No counterpart in the reference, whose cache is bfloat16 or float32 (qwen_wrap.py:68-75); the reads have the semantics
of full_attention (full.py:17-44) and gather_attention (sparse.py:63-67) over the values the codes stand for.
Where a length or start per sequence is a device tensor, nothing is read back to the host, so a captured graph follows
its later values.
"""
from __future__ import annotations

import torch

from . import _native as nat
from . import hip_range
from .hip_attend import HEAD_DIM

BLOCKS = (16, 32, 64)
SMALLEST = 127 - 110   # the scale byte of 2^-110
_POSITIONS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)
_DTYPES = {torch.bfloat16: nat.DT_BF16, torch.float16: nat.DT_F16, torch.float32: nat.DT_F32}


class QuantCache:
    """One layer's K and V in 8 bits: k, v torch.float8_e4m3fn [B,G,C,128]; k_exp, v_exp uint8 [B,G,ceil(C/block)], the
    scale of a block being 2^(x - 127). All four are contiguous tensors on one HIP device, used in place. Scale bytes are 17
    to 247, as quantize_append writes them; those of blocks that hold no row a read takes may be any, but a first write
    that begins inside a block takes the block's byte for that of rows before it (`empty` sets the smallest)."""

    __slots__ = ("k", "v", "k_exp", "v_exp", "block", "batch", "groups", "capacity", "device")

    def __init__(self, k, v, k_exp, v_exp, *, block: int = 64):
        if block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}, got {block!r}")
        shape, device = k.shape, k.device
        B, G, C, d = shape if len(shape) == 4 else (0, 0, 0, 0)
        if d != HEAD_DIM or k.dtype != torch.float8_e4m3fn or not k.is_contiguous() or not k.is_cuda:
            raise ValueError(f"k must be a contiguous float8_e4m3fn [B, G, C, {HEAD_DIM}] tensor on a HIP device")
        if v.shape != shape or v.dtype != torch.float8_e4m3fn or not v.is_contiguous() or v.device != device:
            raise ValueError("v must match k")
        want = torch.Size((B, G, -(-C // block)))
        for t in (k_exp, v_exp):
            if t.shape != want or t.dtype != torch.uint8 or not t.is_contiguous() or t.device != device:
                raise ValueError(f"{'k_exp' if t is k_exp else 'v_exp'} must be a contiguous uint8 {list(want)} tensor on "
                                 f"the cache's device")
        self.k, self.v, self.k_exp, self.v_exp, self.block = k, v, k_exp, v_exp, int(block)
        self.batch, self.groups, self.capacity, self.device = B, G, C, device

    @classmethod
    def empty(cls, batch: int, groups: int, capacity: int, *, block: int = 64, device) -> "QuantCache":
        """A cache with nothing written: codes hold whatever the memory held, which no read of written rows meets, and the
        scales are the smallest, so that a first write inside a block takes the scale it needs."""
        if block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}, got {block!r}")
        if min(int(batch), int(groups), int(capacity)) < 1:
            raise ValueError("batch, groups and capacity must be positive")
        shape = (int(batch), int(groups), int(capacity), HEAD_DIM)
        k, v = (torch.empty(shape, dtype=torch.float8_e4m3fn, device=device) for _ in "kv")
        ke, ve = (torch.full((*shape[:2], -(-shape[2] // block)), SMALLEST, dtype=torch.uint8, device=device) for _ in "kv")
        return cls(k, v, ke, ve, block=block)

    def bytes(self) -> int:
        return sum(t.numel() for t in (self.k, self.v, self.k_exp, self.v_exp))


def _start(cache: QuantCache, start, length: int):
    """(address or None, int) of a start that is an int32 [B] device tensor, or an int, checked here."""
    if isinstance(start, torch.Tensor):
        return hip_range.check_lengths(start, cache.batch, cache.device).data_ptr(), 0
    start = int(start)
    if start < 0 or start + length > cache.capacity:
        raise ValueError(f"rows [{start}, {start + length}) outside the cache's capacity {cache.capacity}")
    return None, start


def _rows(x, step: int):
    """(x as the kernel takes it, its address and three outer strides): unit stride along a row and 16-byte aligned rows of
    `step` elements to 16 bytes (a copy where it has neither). A dimension of one position has no stride: torch may keep
    any there."""
    sb, sg, st, sd = x.stride()
    at = x.data_ptr()
    if sd != 1 or (sb | sg | st) % step or at % 16:
        sb, sg, st = (0 if n == 1 else s for n, s in zip(x.shape[:3], (sb, sg, st)))
        if sd != 1 or (sb | sg | st) % step or at % 16:
            x = x.clone(memory_format=torch.contiguous_format)   # contiguous() is x itself where only its address is odd
            sb, sg, st, _ = x.stride()
            at = x.data_ptr()
    return x, at, sb, sg, st


def _check_rows(cache: QuantCache, k, v):
    """(dtype code, T) of the rows k, v [B,G,T,128] of a write."""
    shape = k.shape
    B, G, T, d = shape if len(shape) == 4 else (0, 0, 0, 0)
    if B != cache.batch or G != cache.groups or d != HEAD_DIM or v.shape != shape:
        raise ValueError(f"k and v must be [B, G, T, {HEAD_DIM}] with B, G = {cache.batch}, {cache.groups}, got "
                         f"{tuple(shape)} and {tuple(v.shape)}")
    dtype = _DTYPES.get(k.dtype)
    if dtype is None or v.dtype != k.dtype:
        raise ValueError(f"k and v must both be bfloat16, float16 or float32, got {k.dtype} and {v.dtype}")
    if k.device != cache.device or v.device != cache.device:
        raise ValueError("k and v must live on the cache's device")
    return dtype, T


def quantize_append(cache: QuantCache, k, v, start=0) -> None:
    """Write the rows k, v [B,G,T,128] (bfloat16, float16 or float32, any strides) at positions [start, start + T).

    start: an int, or an int32 [B] device tensor with each sequence's own (rows outside [0, capacity) are then not
    written). Every block's scale is the smallest power of two, 2^-110 at least, that its rows fit under; a block that
    already holds rows before `start` keeps its scale unless a new row needs a larger one, and then its earlier codes
    are moved to it. So a chunked write may round a value below 2^-6 of its scale twice where one write would round it
    once; everything else is the same. Rows at and after start + T are no longer valid rows of the block they share, but a
    block that grew for rows since discarded keeps that scale and rounding (qwen_wrap.LabCache.rollback undoes it).
    NaN and infinity become NaN; finite values past 1.875 * 2^127 saturate.
    """
    dtype, T = _check_rows(cache, k, v)
    device = cache.device
    starts, at = _start(cache, start, T)
    step = 4 if dtype == nat.DT_F32 else 8
    k, k_at, kb, kg, kt = _rows(k, step)
    v, v_at, vb, vg, vt = _rows(v, step)
    nat.call_on(device, "attnlab_quant_append", k_at, kb, kg, kt, v_at, vb, vg, vt, dtype, cache.k.data_ptr(),
                cache.v.data_ptr(), cache.k_exp.data_ptr(), cache.v_exp.data_ptr(), starts, at, cache.batch, cache.groups, T,
                cache.capacity, cache.block, nat.stream_of(device))


class KeptRows:
    """The last R rows written to a cache as they came: position p in slot p % R of k, v (bfloat16 [B,G,R,128], contiguous).
    What a cache that takes rows back writes them again from."""

    __slots__ = ("cache", "k", "v", "rows")

    def __init__(self, cache: QuantCache, k, v):
        self.cache, self.k, self.v, self.rows = cache, k, v, int(k.shape[2]) if k.dim() == 4 else 0
        for t in (k, v):
            if tuple(t.shape) != (cache.batch, cache.groups, self.rows, HEAD_DIM) or t.dtype != torch.bfloat16 \
                    or not t.is_contiguous() or t.device != cache.device or not self.rows:
                raise ValueError(f"kept rows must be two contiguous bfloat16 [{cache.batch}, {cache.groups}, R, {HEAD_DIM}] "
                                 f"tensors of R >= 1 on the cache's device")


def append_kept(kept: KeptRows, k, v, start: int) -> None:
    """quantize_append of bfloat16 rows to the kept rows' cache; the last of them are kept too."""
    cache = kept.cache
    dtype, T = _check_rows(cache, k, v)
    if dtype != nat.DT_BF16:
        raise ValueError(f"rows to keep must be bfloat16, got {k.dtype}")
    _, at = _start(cache, int(start), T)
    k, k_at, kb, kg, kt = _rows(k, 8)
    v, v_at, vb, vg, vt = _rows(v, 8)
    nat.call_on(cache.device, "attnlab_quant_append_kept", k_at, kb, kg, kt, v_at, vb, vg, vt, cache.k.data_ptr(),
                cache.v.data_ptr(), cache.k_exp.data_ptr(), cache.v_exp.data_ptr(), at, cache.batch, cache.groups, T,
                cache.capacity, cache.block, kept.k.data_ptr(), kept.v.data_ptr(), kept.rows, nat.stream_of(cache.device))


def dequantize_rows(cache: QuantCache, start=0, length=None, *, dtype=torch.bfloat16):
    """The values of positions [start, start + length) -> (k, v), each [B,G,length,128] in `dtype` (bfloat16 and float32
    exact, float16 rounded). start: an int, or an int32 [B] device tensor (positions outside the cache then give zeros;
    length is required). length None: to the capacity."""
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    if length is None:
        if isinstance(start, torch.Tensor):
            raise ValueError("a start per sequence needs a length")
        length = cache.capacity - int(start)
    T = int(length)
    if T < 0:
        raise ValueError(f"length={T} must not be negative")
    starts, at = _start(cache, start, T)
    B, G, device = cache.batch, cache.groups, cache.device
    k = torch.empty((B, G, T, HEAD_DIM), dtype=dtype, device=device)
    v = torch.empty_like(k)
    nat.call_on(device, "attnlab_quant_read", cache.k.data_ptr(), cache.v.data_ptr(), cache.k_exp.data_ptr(),
                cache.v_exp.data_ptr(), k.data_ptr(), v.data_ptr(), code, starts, at, B, G, T, cache.capacity, cache.block,
                nat.stream_of(device))
    return k, v


def quant_attention(q, cache: QuantCache, *, valid_length=None, query_start=None, window=None, sinks: int = 0,
                    scale=None, out=None, out_dtype=torch.bfloat16, partitions=None):
    """Attention of q [B,G,h,T,128] (bfloat16) over an 8-bit cache -> [B,G,h,T,128].

    The T queries sit at consecutive positions from query_start (default: the last T legal ones); query at p reads
    positions j <= p, j < valid_length, and with a window j > p - window or j < sinks. Sums are fp32 under weights of at
    most 1: n rows of values below 2^128 / n have finite outputs. valid_length: an int (default:
    the capacity), or for one query an int32 [B] device tensor with each sequence's length, clamped to [0, capacity],
    its query at the last position. A query that reads no position gets zeros. One query takes h <= 8 at every form and
    out_dtype float32 too, with weights of 16 bits; a chunk, and one query with h <= 16 and an int length, gives bfloat16, and
    rounds its weights to bfloat16 before their product with V (2^-8 of each at most; their sum is not rounded). partitions
    overrides the split-K count (one query: 1..256, a chunk: 1..16).
    """
    return hip_range.range_attention(q, cache.k.data_ptr(), cache.v.data_ptr(),
                                     (cache.k_exp.data_ptr(), cache.v_exp.data_ptr()), cache.block, cache.batch,
                                     cache.groups, cache.capacity, cache.device, valid_length, query_start, window, sinks,
                                     scale, out, out_dtype, partitions)


def quant_gather_attention(q, cache: QuantCache, selected, selected_valid=None, *, scale=None, out=None,
                           out_dtype=torch.bfloat16, partitions=None):
    """gather_attention over an 8-bit cache: q [B,G,h,1,128] over the listed positions selected [B,G,S] (signed
    integers or uint8), read in place. Slots with selected_valid False, and positions outside [0, capacity), are skipped;
    a position listed twice counts twice; a query with no row gets zeros."""
    if selected.dim() != 3 or tuple(selected.shape[:2]) != (cache.batch, cache.groups) \
            or selected.dtype not in _POSITIONS:
        raise ValueError(f"selected must be an integer [B, G, S] tensor with B, G = {cache.batch}, {cache.groups}, got "
                         f"{selected.dtype} {tuple(selected.shape)}")
    if selected.device != cache.device:
        raise ValueError("selected must live on the cache's device")
    if selected_valid is not None and selected_valid.shape != selected.shape:
        raise ValueError("selected_valid must match selected")
    if selected.dtype == torch.int64:   # a position past 32 bits is outside the cache, not another one
        selected = selected.clamp(-1, cache.capacity)
    selected = selected.to(torch.int32)   # before the -1 of the slots to skip, which unsigned types do not hold
    if selected_valid is not None:
        selected = torch.where(selected_valid.bool(), selected, -1)
    return hip_range.listed_attention(q, cache, selected.contiguous(), scale=scale, out=out, out_dtype=out_dtype,
                                      partitions=partitions)
