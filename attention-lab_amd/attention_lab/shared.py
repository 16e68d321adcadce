"""Attention of sequences that share long prompts, over a paged cache: a prompt's keys and values are read once for all the
sequences that continue it, where attend_paged reads them once for each.

Beside hip_attend.attend_paged and pages.py, whose forks are what shares pages. The full read's semantics (full.py:17-44) over
each sequence's own table; no counterpart in the reference, whose caches are contiguous.
"""
from __future__ import annotations

import torch

from . import _native as nat
from .hip_attend import HEAD_DIM
from .hip_range import DEFAULT_SCALE, INT_MAX, MAX_H_CHUNK, aligned_query, check_lengths, check_out

WIDE_ROWS, NARROW_ROWS = 128, 16   # (query, head) rows of a workgroup of either kernel
MAX_SPLITS = 64
PART_BYTES = 132 * 4               # of a row's partial


def shared_splits(G: int, rows: int, wide: bool, chunk: bool = False) -> int:
    """Partials of the shared part that a row's room is made for, `rows` (query, head) rows of a group over all sequences: the
    workgroups that come to a tile of rows if all sequences share, and a piece (chunk: several queries a sequence)."""
    per, workers = (NARROW_ROWS, 768) if not wide else (WIDE_ROWS, 512 if chunk else 256)
    return min(MAX_SPLITS, workers // (G * -(-rows // per)) + 2)


def own_splits(BG: int, rows: int, keys: int) -> int:
    """Key splits of the own part: `rows` rows of each of BG (sequence, group) pairs over up to `keys` positions. 384 narrow
    workgroups; with 192 and 768: 2 x 8 answers of 2K behind 2K 42 and 36 us for 33, 16 answers of 300 behind 8K 27 and 32 for
    27."""
    wide = rows > MAX_H_CHUNK
    tiles = BG * -(-rows // (WIDE_ROWS if wide else NARROW_ROWS))
    return max(1, min(16, (512 if wide else 384) // tiles, keys // 256))


def _lengths(x, n: int, device, name: str):
    """(address or None, int) of a value per sequence or run on the device, or one for all."""
    if isinstance(x, torch.Tensor):
        return check_lengths(x, n, device).data_ptr(), 0
    x = int(x)
    if not 0 <= x <= INT_MAX:
        raise ValueError(f"{name}={x} must be in [0, 2^31)")
    return None, x


def shared_prefix_attention(q, k_pages, v_pages, block_table, lengths, prefix_lengths=0, *, runs=None, scale=None, out=None,
                            partitions=None):
    """q [B,G,h,T,128] bfloat16, k_pages and v_pages bfloat16 [num_pages,G,page_size,128] (page_size a power of two),
    block_table int32 [B,max_pages] -> bfloat16 [B,G,h,T,128].

    Sequence b's T queries sit at the last positions of lengths[b] (an int for all, or int32 [B] on the device; clamped to
    max_pages * page_size) and read positions j up to their own by its table; positions on an entry outside [0, num_pages) are
    skipped, and a query that reads nothing gets zeros. h <= 16.

    Sequences runs[r] .. runs[r + 1] - 1 (runs int32 [R + 1] on the device, ascending; None: one run of all) share their first
    prefix_lengths[r] positions (an int for all, or int32 [R] on the device): below it, rounded down to whole pages, the
    tables of those that are long enough for all of their queries to see the whole prefix name the same pages, and one's are
    read for all. The others, and sequences in no run, read everything by their own tables. prefix_lengths 0: a read of a paged
    cache with a length per sequence.

    Nothing is read back to the host, so a captured graph follows the tensors' later values. One query's weights keep 16 bits in
    their product with V; a chunk's (T > 1) are rounded to bfloat16 before it (2^-8 of each at most). Their sum is not rounded,
    sums are float32. An infinite value that a query sees makes its output NaN or infinite. There is no gradient: tensors that
    ask for one are refused. partitions overrides how
    many partials a row may have of the shared part (1 to 64; 0: the prefix is ignored) and of the own one (1 to 64)."""
    pool, device = k_pages.shape, k_pages.device
    if (len(pool) != 4 or pool[3] != HEAD_DIM or k_pages.dtype is not torch.bfloat16 or not k_pages.is_contiguous()
            or not k_pages.is_cuda):
        raise ValueError(f"k_pages must be a contiguous bfloat16 [num_pages, G, page_size, {HEAD_DIM}] pool on a HIP device")
    if v_pages.shape != pool or v_pages.dtype is not torch.bfloat16 or not v_pages.is_contiguous() or v_pages.device != device:
        raise ValueError("v_pages must match k_pages")
    pages, G, page, _ = pool
    shape = q.shape
    if len(shape) != 5 or shape[1] != G or shape[4] != HEAD_DIM or q.dtype is not torch.bfloat16 or q.device != device:
        raise ValueError(f"q must be a bfloat16 [B, {G}, h, T, {HEAD_DIM}] tensor on the pools' device, got {q.dtype} "
                         f"{tuple(shape)}")
    B, _, h, T, _ = shape
    if not 1 <= h <= MAX_H_CHUNK:
        raise ValueError(f"h={h} must be in [1, {MAX_H_CHUNK}]")
    if B < 1 or not pages or not G or not page or page & (page - 1):
        raise ValueError("need at least one sequence, page and group, and a page_size that is a power of two, got "
                         f"{B}, {pages}, {G}, {page}")
    rows_b, W = block_table.shape if block_table.dim() == 2 else (0, 0)
    if rows_b != B or W < 1 or block_table.dtype is not torch.int32 or block_table.device != device:
        raise ValueError("block_table must be an int32 [B, max_pages] tensor with unit column stride on the pools' device")
    step, unit = block_table.stride()
    if unit != 1 and W > 1:
        raise ValueError("block_table must be an int32 [B, max_pages] tensor with unit column stride on the pools' device")
    R = 1
    if runs is not None:
        R = runs.numel() - 1
        if runs.dim() != 1 or R < 1 or runs.dtype is not torch.int32 or not runs.is_contiguous() or runs.device != device:
            raise ValueError("runs must be a contiguous int32 [R + 1] tensor of at least two bounds on the pools' device")
    nat.refuse_gradients("shared_prefix_attention", q, k_pages, v_pages)
    lengths_at, length = _lengths(lengths, B, device, "lengths")
    prefix_at, prefix = _lengths(prefix_lengths, R, device, "prefix_lengths")
    most = W * page if lengths_at else min(length, W * page)
    keys = most if prefix_at else min(prefix, most) // page * page
    q, q_at = aligned_query(q)
    out = check_out(out, q, torch.bfloat16)
    if T == 0:
        return out
    rows = B * h * T
    # Tiles of 128 rows from half a narrow one on (us, wide and narrow: 16 runs of 16 rows on 4K 58 and 71, 32 of 8 rows 101 and
    # 92; one run on 4K of 8 rows 19.0 and 18.3, of 16 rows 19.2 and 19.4, of 64 rows 22 and 26)
    wide = T > 1 or 2 * rows > NARROW_ROWS * R
    if partitions is None:
        ns = shared_splits(G, rows, wide, T > 1) if keys else 0
        no = own_splits(B * G, h * T if T > 1 else 1, most if prefix_at else most - keys)
    else:
        ns, no = (int(x) for x in partitions)
        if not (0 <= ns <= MAX_SPLITS and 1 <= no <= MAX_SPLITS):
            raise ValueError(f"partitions must be two counts, in [0, {MAX_SPLITS}] and [1, {MAX_SPLITS}]")
    rows *= G
    nbytes = ((rows + 1) // 2 * 16 + rows * (ns + no) * PART_BYTES) if ns + no > 1 else 0   # attnlab_shared_part_bytes
    part = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    nat.call_on(device, "attnlab_shared_prefix_attend", q_at, k_pages.data_ptr(), v_pages.data_ptr(), pages, page,
                block_table.data_ptr(), max(step, W) if B == 1 else step, W, lengths_at, length,
                prefix_at, prefix, nat.ptr(runs), R, B, G, h, T, DEFAULT_SCALE if scale is None else float(scale), wide, ns, no,
                out.data_ptr(), nat.ptr(part), nbytes, nat.stream_of(device))
    return out
