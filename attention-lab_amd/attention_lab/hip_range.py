"""Attention over a range of a cache on gfx950: every legal position, or a sliding window and a few first ones (sinks),
for one query or a causal chunk, over a bfloat16 cache or an 8-bit one; and the row-list read of an 8-bit cache.

The kernels behind `window_attention` (window.py) and `quant_attention` / `quant_gather_attention` (quant.py), which
check their caches; this module checks what the reads share, chooses the split counts and launches, on the tensors' own
device and torch's current stream of it.

The last workgroup of a (b, g) to arrive merges its split-K partials where a counter tells it that it is: the counters
and partials of such single launches belong to a stream (4.3 MB each, held for the process's life), whose launches follow one
another and leave the counters zero.
Other calls, a captured one among them, allocate partials of their own and take a second launch for the merge (the same
sums), so a graph shares nothing with other graphs or calls.
"""
from __future__ import annotations

import math

import torch

from . import _native as nat
from .hip_attend import HEAD_DIM

MAX_H = 8           # query heads per KV group of the one-query kernels (the matrix core's 16 columns hold each twice)
MAX_H_CHUNK = 16    # ... of the chunk kernel
CHUNK_ROWS = 128    # (query, head) rows of the chunk kernel's workgroup
CHUNK_KEYS = 64     # keys of its block
TILE = 32           # rows a wave of the one-query kernel takes at a time
MAX_SPLITS = 16
MAX_P = 256
MERGE_SLOTS = 16    # partials the last workgroup to arrive merges itself; more take a second launch
INT_MAX = 2 ** 31 - 1
DEFAULT_SCALE = 1.0 / math.sqrt(HEAD_DIM)


def decode_partitions(BG: int, count: int, ragged: bool = False, listed: bool = False) -> int:
    """Split-K count of the one-query kernels for BG (b, g) rows of `count` positions each: one workgroup per CU, or two
    where that leaves one more than a seventh of the CUs idle or each of two 48 tiles of 32 positions; and at least two
    tiles for every one of a workgroup's four waves (one of listed rows). Measured on MI355X (graph replay, 8-bit), one
    per CU against two: BG=8 at 8K 10.3 / 11.9 us, at 64K 27.6 / 31.9; BG=32 at 16K 27.8 / 31.0; BG=64 at 8K 27.5 /
    30.0, at 12K 38.8 / 38.2, at 20K 55.6 / 54.6; BG=128 at 32K 162 / 158; BG=56 (224 workgroups of one) at 4K 17.3 /
    18.3; BG=96 (192) at 4K 25.9 / 23.0; BG=160 (160) at 2K 25.8 / 21.4. Two tiles a wave against one: BG=8 at 2K 8.2 /
    9.1, at 512 7.2 / 7.3; of 1092 listed rows, BG=16, 12.0 / 11.5.
    ragged (a length per sequence, `count` by the capacity): the slots that the kernel deals out by the sequences'
    lengths, with the half slot that every sequence's remainder takes: two workgroups per CU, or four where two leave a
    tenth of the chip idle; at most one to 128 positions. BG=40 to 20K: 13 slots 30.5 us, 16 35.9; BG=128 to 32K: 4 (448
    of 512 places) 129, 8 (960 of 1024) 122; BG=256 to 2K: 2 31.0, 4 27.2; BG=8 of 2K: 16 9.7, 64 9.9."""
    BG = max(BG, 1)
    if ragged:
        P = (512 + BG // 2) // BG
        if P * BG - BG // 2 < 460:
            P = (1024 + BG // 2) // BG
        return max(2, min(64, P, count // (4 * TILE)))
    P = 256 // BG
    if BG * count >= 512 * 48 * TILE or P * BG < 220:
        P = 512 // BG
    return max(1, min(64, P, count // ((4 if listed else 8) * TILE)))


def chunk_splits(BG: int, h: int, T: int, keys: int) -> int:
    """Workgroups that share a query tile's keys (`keys`: those the longest tile reads). Two workgroups per CU where that
    leaves each 1024 keys or more, else one per CU with at least 320: a share writes and reads back 67 KB of partials,
    and a grid between one and two per CU takes as long as two. MI355X, 8-bit, us for splits of 1, 2, 4, 8: 1000 queries
    (h=2) after 29011, 128 tiles, 549, 290, 250, 256; a 2K prompt (h=2), 256 tiles, 45, 40, 46; a 1K prompt (h=4), 256
    tiles, 27, 33, 41; 200 queries (h=4) after 2500, 56 tiles, 55, 38, 30, 33; 300 (h=3) after 700, 64 tiles, 25, 22, 22,
    28; 512 (h=4) after none, 128 tiles, 16, 22, 26; 1501 under a window of 2047, 384 tiles, 76, 78."""
    tiles = BG * -(-T // (CHUNK_ROWS // h))
    s = min(MAX_SPLITS, 512 // tiles)
    if keys < 1024 * s:
        s = min(MAX_SPLITS, 256 // tiles, keys // 320)
    return max(s, 1)


def check_window(window, sinks):
    """(window, sinks) for the kernels, window 0 for none."""
    sinks = int(sinks)
    if sinks < 0:
        raise ValueError(f"sinks={sinks} must not be negative")
    if window is None:
        return 0, 0
    window = int(window)
    if window < 1:
        raise ValueError(f"window={window} must be at least 1 (None: no window)")
    return min(window, INT_MAX), min(sinks, INT_MAX)


def check_query(q, B: int, G: int, device):
    """q [B,G,h,T,128] bfloat16 on the cache's device -> (h, T)."""
    shape = q.shape
    if len(shape) != 5 or shape[0] != B or shape[1] != G or shape[4] != HEAD_DIM or q.dtype != torch.bfloat16:
        raise ValueError(f"q must be a bfloat16 [B, G, h, T, {HEAD_DIM}] tensor with B, G = {B}, {G}, got {q.dtype} "
                         f"{tuple(shape)}")
    if q.device != device:
        raise ValueError("q must live on the cache's device")
    h = shape[2]
    if not 1 <= h <= MAX_H_CHUNK:
        raise ValueError(f"h={h} must be in [1, {MAX_H_CHUNK}]")
    return h, shape[3]


def aligned_query(q):
    """(q contiguous at a 16-byte aligned address, that address): a copy where it is not."""
    q = q.contiguous()
    at = q.data_ptr()
    if at % 16:
        q = q.clone()
        at = q.data_ptr()
    return q, at


def check_listed(q, B: int, G: int, device, partitions) -> int:
    """q and the split count of a row-list read -> h."""
    h, T = check_query(q, B, G, device)
    if T != 1:
        raise ValueError("the row-list read takes one query position")
    if h > MAX_H:
        raise ValueError(f"the row-list read takes h <= {MAX_H} query heads per group, got {h}")
    split_count(partitions, 1, MAX_P)
    return h


def check_lengths(lengths, B: int, device):
    """A device tensor of one valid length (or start) per sequence."""
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (B,) or not lengths.is_contiguous() \
            or lengths.device != device:
        raise ValueError(f"one value per sequence must be a contiguous int32 [{B}] tensor on the cache's device")
    return lengths


def check_out(out, q, dtype):
    if out is None and dtype is torch.bfloat16:
        # q is contiguous where it stands for the layout: empty_like is half the time of an empty with its arguments
        return torch.empty_like(q)
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("out_dtype must be float32 or bfloat16")
    if out is None:
        return torch.empty_like(q, dtype=dtype)
    if tuple(out.shape) != tuple(q.shape) or out.dtype != dtype or not out.is_contiguous() or out.device != q.device:
        raise ValueError(f"out must be a contiguous {dtype} tensor shaped like q on its device")
    return out


def split_count(partitions, chosen: int, most: int) -> int:
    """The caller's split count, checked, or the rule's."""
    if partitions is None:
        return chosen
    if not 1 <= int(partitions) <= most:
        raise ValueError(f"partitions must be in [1, {most}]")
    return int(partitions)


_MERGES: dict = {}      # (device index, stream) -> its counters, zeroed once and left zero by every call, and partials
COUNTERS = 4096         # (b, g) rows that they serve
PARTIALS = 8 * 1024     # (slot, head) partials: up to four workgroups per CU of eight heads, 4.3 MB
PART_WORDS = HEAD_DIM + 2


def _merge_here(h: int, P: int, positions: int, ragged: bool) -> bool:
    """Whether a call merges in its own launch (P <= MERGE_SLOTS), which spares the host a launch (3.5 us) and, for few
    partials, the GPU up to 1 us. Long reads with many partials merge faster in a launch of their own: h=8, P=16, BG=16 at
    16K 18.6 us for 22.2 (at 4K, BG=8, 10.2 for 12.8, but the host's part is 9 or 12.5); with a length per sequence, whose
    merge is the workgroup's with the most slots, 40 x 20K 30.5 for 32.8, 256 x 2K 31.0 for 30.1."""
    return positions <= 1 << 19 if ragged else h * P <= 64 or positions <= 1 << 17


def stream_counters(device, stream: int):
    """(tensor, address) of a stream's counters, which are zero between launches, and partials behind them."""
    buf = _MERGES.get((device.index, stream))
    if buf is None:
        buf = _MERGES[device.index, stream] = torch.zeros(COUNTERS + PARTIALS * PART_WORDS, dtype=torch.int32, device=device)
    return buf, buf.data_ptr()


def _split_k(P: int, BG: int, h: int, device, stream: int, counted: bool):
    """(tensor to hold on to, partials' address, counters' address) of a one-query call split over P workgroups."""
    if P == 1:
        return None, None, None
    rows = BG * P * h
    if counted and P <= MERGE_SLOTS and BG <= COUNTERS and rows <= PARTIALS and not capturing(device):
        buf, at = stream_counters(device, stream)
        return buf, at + 4 * COUNTERS, at
    part = torch.empty(rows * PART_WORDS, dtype=torch.float32, device=device)
    return part, part.data_ptr(), None


def capturing(device) -> bool:
    """torch's current stream on `device` is being captured."""
    if device.index == torch._C._cuda_getDevice():
        return torch._C._cuda_isCurrentStreamCapturing()
    with torch.cuda.device(device):
        return torch._C._cuda_isCurrentStreamCapturing()


# The host's part of a call is most of a small one's time, so the checks below look only at what the call gives.
def range_attention(q, k_ptr: int, v_ptr: int, exp_ptrs, block: int, B: int, G: int, C: int, device, valid_length,
                    query_start, window, sinks, scale, out, out_dtype, partitions):
    """The reads of window_attention and quant_attention over a checked cache [B,G,C,128] at k_ptr / v_ptr (exp_ptrs: the
    scale bytes of an 8-bit one, or (None, None))."""
    if not (B and G and C):
        raise ValueError(f"the cache must hold at least one sequence, group and position, got {B}, {G}, {C}")
    h, T = check_query(q, B, G, device)
    if window is not None or sinks:
        window, sinks = check_window(window, sinks)
    else:
        window = sinks = 0
    lengths = None
    if isinstance(valid_length, torch.Tensor):
        lengths = check_lengths(valid_length, B, device).data_ptr()
        if T != 1 or query_start is not None:
            raise ValueError("a length per sequence goes with one query each, at its sequence's last position")
        if h > MAX_H:
            raise ValueError(f"a length per sequence takes h <= {MAX_H} query heads per group, got {h}")
        legal, p0, seen = C, C - 1, C
    else:
        legal = C if valid_length is None else int(valid_length)
        if not 0 < legal <= C:
            raise ValueError(f"valid_length={legal} must be in (0, capacity={C}]")
        p0 = legal - T if query_start is None else int(query_start)
        if not 0 <= p0 < INT_MAX - T:
            raise ValueError(f"query positions must be non-negative and below 2^31, got {p0}")
        seen = legal if query_start is None else min(legal, p0 + T)
    if window:   # what the query, or a chunk's workgroup, reads
        seen = min(seen, window + min(T, CHUNK_ROWS // h) - 1 + min(sinks, seen))
    q, q_at = aligned_query(q)
    sc = DEFAULT_SCALE if scale is None else float(scale)
    stream = nat.stream_of(device)
    if T == 1 and h <= MAX_H:
        out = check_out(out, q, out_dtype)
        P = decode_partitions(B * G, seen, lengths is not None) if partitions is None else split_count(partitions, 1, MAX_P)
        held, part, arrive = _split_k(P, B * G, h, device, stream, _merge_here(h, P, B * G * seen, lengths is not None))
        nat.call_on(device, "attnlab_range_decode", k_ptr, v_ptr, *exp_ptrs, block, q_at, lengths, legal, p0, window,
                    sinks, B, G, h, C, P, sc, out.data_ptr(), out_dtype == torch.bfloat16, part, arrive, stream)
        return out
    if out_dtype != torch.bfloat16:
        raise ValueError("a chunk's outputs are bfloat16")
    out = check_out(out, q, out_dtype)
    if T == 0:
        return out
    splits = chunk_splits(B * G, h, T, seen) if partitions is None else split_count(partitions, 1, MAX_SPLITS)
    nbytes, part = 0, None
    if splits > 1:
        nbytes = nat.lib().attnlab_range_prefill_part_bytes(B, G, h, T, splits)
        held = torch.empty(nbytes // 4, dtype=torch.float32, device=device)
        part = held.data_ptr()
    nat.call_on(device, "attnlab_range_prefill", q_at, k_ptr, v_ptr, *exp_ptrs, block, out.data_ptr(), B, G, h, T,
                p0, legal, C, window, sinks, sc, splits, part, nbytes, stream)
    return out


def listed_attention(q, cache, rows, *, scale, out, out_dtype, partitions):
    """The row-list read of quant_gather_attention: rows int32 [B,G,S] contiguous, checked cache."""
    B, G, C, device = cache.batch, cache.groups, cache.capacity, cache.device
    h = check_listed(q, B, G, device, partitions)
    S = int(rows.shape[2])
    if S < 1:
        raise ValueError("at least one row must be selected")
    q, q_at = aligned_query(q)
    out = check_out(out, q, out_dtype)
    P = split_count(partitions, decode_partitions(B * G, S, listed=True), MAX_P)
    stream = nat.stream_of(device)
    held, part, arrive = _split_k(P, B * G, h, device, stream, _merge_here(h, P, B * G * S, False))
    sc = DEFAULT_SCALE if scale is None else float(scale)
    nat.call_on(device, "attnlab_quant_attend", cache.k.data_ptr(), cache.v.data_ptr(), cache.k_exp.data_ptr(),
                cache.v_exp.data_ptr(), cache.block, q_at, rows.data_ptr(), S, B, G, h, S, C, P, sc,
                out.data_ptr(), int(out_dtype == torch.bfloat16), part, arrive, stream)
    return out
