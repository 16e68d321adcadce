"""Attention with a sliding window and a few first positions that stay visible (sinks), over the bfloat16 cache.

The fixed set F of the selection rule (selection.py) read as a range, at any size: `window_attention(..., window=64,
sinks=4)` of one query reads F. The same mask over an 8-bit cache is quant.quant_attention(window=, sinks=).
"""
from __future__ import annotations

import torch

from . import hip_range
from .hip_attend import HEAD_DIM
from .selection import FIXED_PREFIX


def window_attention(q, k, v, *, window, sinks: int = FIXED_PREFIX, valid_length=None, query_start=None, scale=None,
                     out=None, out_dtype=torch.bfloat16, partitions=None):
    """q [B,G,h,T,128], k, v [B,G,C,128] (bfloat16, k and v contiguous) -> [B,G,h,T,128].

    The T queries sit at consecutive positions from query_start (default: the last T legal ones); query at p reads
    positions j <= p, j < valid_length with j > p - window or j < sinks, by their original positions. window None:
    every legal position. Sums are fp32 under weights of at most 1: n rows of values below 2^128 / n have finite outputs.
    valid_length: an int (default: the capacity), or for one query an int32 [B] device tensor
    with each sequence's length, clamped to [0, C], its query at the last position. A query that reads no position
    gets zeros. One query takes h <= 8 at every form and out_dtype float32 too, with weights of 16 bits; a chunk, and one
    query with h <= 16 and an int length, gives bfloat16, and rounds its weights to bfloat16 before their product with V (2^-8
    of each at most; their sum is not rounded). partitions overrides the split-K count (one query: 1..256, a chunk: 1..16).
    """
    if k.dim() != 4 or k.shape[3] != HEAD_DIM or k.dtype != torch.bfloat16 or not k.is_contiguous() or not k.is_cuda:
        raise ValueError(f"the cache must be a contiguous bfloat16 [B, G, C, {HEAD_DIM}] tensor on a HIP device")
    if v.shape != k.shape or v.dtype != k.dtype or not v.is_contiguous() or v.device != k.device:
        raise ValueError("v must match k")
    B, G, C, _ = k.shape
    return hip_range.range_attention(q, k.data_ptr(), v.data_ptr(), (None, None), 0, B, G, C, k.device, valid_length,
                                     query_start, window, sinks, scale, out, out_dtype, partitions)
