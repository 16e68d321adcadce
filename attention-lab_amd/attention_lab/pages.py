"""A K/V cache in pages that sequences share: branching, making room, writing, shortening and compacting, on gfx950.

A `PagedCache` holds the K and V of several layers in pools of pages, and which pages a sequence's positions are in. A page
can belong to many sequences, so a prompt with several continuations is held once:

    cache = PagedCache.empty(layers, slots, groups, num_pages, page_size, max_pages, device=dev)
    page_reserve(cache, tokens)                       # slot 0: a prompt of tokens[0] positions, the others 0
    page_append(cache, layer, k, v, tokens)           # every layer's rows
    page_fork(cache, parents)                         # parents all 0: every slot goes on from the prompt
    page_reserve(cache, 1)                            # a next position for each; a page that several would write is copied
    page_append(cache, layer, k, v)
    out = shared_prefix_attention(q, cache.k[layer], cache.v[layer], cache.table, cache.lengths, prompt)   # shared.py
    page_fork(cache, parents)                         # a beam's step: the ones that go on, some of them twice
    page_truncate(cache, lengths)                     # a draft's rejected tokens, or (0) a sequence that has ended
    page_compact(cache)                               # the pages in use to the pool's low end

The pools are those that hip_attend.attend_paged reads. All of it is decided on the device: nothing is read back to the host,
so a captured graph follows the tensors' later values, and the results depend on the cache alone, never on timing. Calls on
one cache must be ordered on one stream. No counterpart in the reference, whose caches are branched by copying them
(qwen_wrap.py:117-133).
"""
from __future__ import annotations

import torch

from . import _native as nat
from .hip_attend import HEAD_DIM
from .quant import _rows

MAX_SLOTS = 1024
MAX_PAGE = 1 << 16
INT_MAX = 2 ** 31 - 1


def _check_book(t, name: str, shape: tuple, device):
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous int32 {list(shape)} tensor on the cache's device")
    return t


class PagedCache:
    """K and V of `layers` layers in pages, for up to 1024 sequence slots.

    k, v bfloat16 [layers, num_pages, G, page_size, 128]; table int32 [slots, max_pages], the page of each slot's positions
    [e page_size, (e + 1) page_size) in its entry e, or -1; lengths int32 [slots]; refs int32 [num_pages], how many entries name
    each page (0: free). All are contiguous tensors on one HIP device, used in place. The operators keep refs in step with the
    table; a table made elsewhere has to come with its counts and hold -1 past its sequences' pages (entries below -1 are the
    operators' own, see page_reserve). A page whose count is raised
    by hand stays in use and is never written in place (a compaction may move it). missing (int32 [1], optional) counts the
    pages that page_reserve could not give."""

    __slots__ = ("k", "v", "table", "lengths", "refs", "missing", "layers", "num_pages", "groups", "page_size", "slots",
                 "max_pages", "layer_bytes", "device")

    def __init__(self, k, v, table, lengths, refs, *, missing=None):
        shape, device = k.shape, k.device
        if len(shape) != 5 or shape[4] != HEAD_DIM or k.dtype != torch.bfloat16 or not k.is_contiguous() or not k.is_cuda:
            raise ValueError(f"k must be a contiguous bfloat16 [layers, num_pages, G, page_size, {HEAD_DIM}] tensor on a HIP "
                             "device")
        if v.shape != shape or v.dtype != k.dtype or not v.is_contiguous() or v.device != device:
            raise ValueError("v must match k")
        layers, pages, G, page, _ = shape
        if not (layers and pages and G and page):
            raise ValueError(f"the pools must hold at least one layer, page, group and row, got {tuple(shape)}")
        if table.dim() != 2 or not 1 <= table.shape[0] <= MAX_SLOTS or table.shape[1] < 1:
            raise ValueError(f"table must be [slots, max_pages] with 1 to {MAX_SLOTS} slots and at least one page, got "
                             f"{tuple(table.shape)}")
        S, W = table.shape
        _check_geometry(pages, G, page, S, W)
        self.table = _check_book(table, "table", (S, W), device)
        self.lengths = _check_book(lengths, "lengths", (S,), device)
        self.refs = _check_book(refs, "refs", (pages,), device)
        self.missing = None if missing is None else _check_book(missing, "missing", (1,), device)
        if (k.data_ptr() | v.data_ptr()) % 16:
            raise ValueError("k and v must be 16-byte aligned")
        self.k, self.v, self.device = k, v, device
        self.layers, self.num_pages, self.groups, self.page_size = int(layers), int(pages), int(G), int(page)
        self.slots, self.max_pages = int(S), int(W)
        self.layer_bytes = 2 * self.num_pages * self.groups * self.page_size * HEAD_DIM   # of K, or of V

    @classmethod
    def empty(cls, layers: int, slots: int, groups: int, num_pages: int, page_size: int, max_pages: int, *,
              device) -> "PagedCache":
        """A cache of empty slots: no page in use, the pools' contents whatever the memory held."""
        layers, slots, groups, num_pages, page_size, max_pages = (int(x) for x in (layers, slots, groups, num_pages, page_size,
                                                                                   max_pages))
        if min(layers, slots, groups, num_pages, page_size, max_pages) < 1 or slots > MAX_SLOTS:
            raise ValueError(f"layers, slots (at most {MAX_SLOTS}), groups, num_pages, page_size and max_pages must be positive")
        _check_geometry(num_pages, groups, page_size, slots, max_pages)
        k, v = (torch.empty(layers, num_pages, groups, page_size, HEAD_DIM, dtype=torch.bfloat16, device=device) for _ in "kv")
        table = torch.full((slots, max_pages), -1, dtype=torch.int32, device=device)
        lengths, refs, missing = (torch.zeros(n, dtype=torch.int32, device=device) for n in (slots, num_pages, 1))
        return cls(k, v, table, lengths, refs, missing=missing)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.table, self.lengths, self.refs))


def _check_geometry(pages: int, G: int, page: int, S: int, W: int) -> None:
    if page & (page - 1) or page > MAX_PAGE:
        raise ValueError(f"page_size must be a power of two up to {MAX_PAGE}, got {page}")
    if W * page > INT_MAX or pages * G * page > INT_MAX or S * W > INT_MAX:
        raise ValueError(f"max_pages * page_size, num_pages * G * page_size and slots * max_pages must be below 2^31, got "
                         f"{W} * {page}, {pages} * {G} * {page} and {S} * {W}")


def _per_slot(cache: PagedCache, x, name: str):
    """(address or None, int) of a value per slot on the device, or one for all."""
    if isinstance(x, torch.Tensor):
        return _check_book(x, name, (cache.slots,), cache.device).data_ptr(), 0
    x = int(x)
    if not 0 <= x <= INT_MAX:
        raise ValueError(f"{name}={x} must be in [0, 2^31)")
    return None, x


def _scratch(cache: PagedCache):
    """Scratch of one call (attnlab_page_scratch_bytes): from torch's allocator, so that a captured graph has its own."""
    nbytes = 16 + 12 * max(cache.slots, cache.num_pages)
    return torch.empty(nbytes, dtype=torch.uint8, device=cache.device), nbytes


def page_fork(cache: PagedCache, parents) -> None:
    """Slot i goes on from what slot parents[i] held before the call (int32 [slots], on the device): it shares its pages and
    has its length. parents is a tensor of its own, not one of the cache's. A parent outside [0, slots) leaves the slot empty.
    Pages that nobody holds any more are free; no K/V row is copied before page_reserve."""
    parents = _check_book(parents, "parents", (cache.slots,), cache.device)
    nat.call_on(cache.device, "attnlab_page_fork", cache.table.data_ptr(), cache.lengths.data_ptr(), cache.refs.data_ptr(),
                parents.data_ptr(), cache.slots, cache.max_pages, cache.num_pages, nat.stream_of(cache.device))


def page_reserve(cache: PagedCache, tokens=1) -> None:
    """Room for `tokens` more positions of every slot (an int, or int32 [slots] on the device; 0 leaves a slot as it is):
    lengths grow by as many (to 2^31 - 1 at most, where rows are no longer written), and page_append may write their rows.

    A slot that ends inside a page that others hold too gets a page of its own, with the page's rows up to its length copied
    in every layer; if all of a page's holders are written to, the last of them keeps it. New pages are the lowest free ones, in
    the order of slots and positions. Where none is left an entry is -1: its positions are neither written nor read (nor those
    past max_pages * page_size), and cache.missing counts it. Where none is left for a page of a slot's own, the slot's rows
    of the shared one stay its own, but neither they nor the new ones are read until page_truncate takes the slot back to
    them (or before): the entry is below -1 till then. One of the slots that would need a copy, the one with the most rows
    in the page, writes on in it if every other one is left so or has its copy."""
    at, each = _per_slot(cache, tokens, "tokens")
    scratch, nbytes = _scratch(cache)
    nat.call_on(cache.device, "attnlab_page_reserve", cache.k.data_ptr(), cache.v.data_ptr(), cache.layers, cache.num_pages,
                cache.groups, cache.page_size, cache.table.data_ptr(), cache.lengths.data_ptr(), cache.refs.data_ptr(), at, each,
                cache.slots, cache.max_pages, nat.ptr(cache.missing), scratch.data_ptr(), nbytes, nat.stream_of(cache.device))


def page_append(cache: PagedCache, layer: int, k, v, tokens=None) -> None:
    """A layer's rows k, v bfloat16 [slots, G, T, 128] (any strides) at the last positions of every slot: row t of slot i at
    lengths[i] - tokens[i] + t for t < tokens[i] (int32 [slots] on the device, what page_reserve was given; None: T for all).
    Rows of a page that another slot holds are its rows too: page_reserve sees to it that there are none. k and v lie in memory that
    the call does not write. There is no gradient: rows that ask for one are refused."""
    shape, device = k.shape, cache.device
    S, G, T, d = shape if len(shape) == 4 else (0, 0, 0, 0)
    if S != cache.slots or G != cache.groups or d != HEAD_DIM or k.dtype is not torch.bfloat16:
        raise ValueError(f"k must be a bfloat16 [slots, G, T, {HEAD_DIM}] tensor with slots, G = {cache.slots}, {cache.groups}, "
                         f"got {k.dtype} {tuple(shape)}")
    if v.shape != shape or v.dtype is not torch.bfloat16 or k.device != device or v.device != device:
        raise ValueError("v must match k, on the cache's device")
    nat.refuse_gradients("page_append", k, v)
    layer = int(layer)
    if not 0 <= layer < cache.layers:
        raise ValueError(f"layer {layer} outside [0, {cache.layers})")
    at = None if tokens is None else _check_book(tokens, "tokens", (S,), device).data_ptr()
    k, k_at, kb, kg, kt = _rows(k, 8)
    v, v_at, vb, vg, vt = _rows(v, 8)
    step = layer * cache.layer_bytes
    nat.call_on(device, "attnlab_page_append", k_at, kb, kg, kt, v_at, vb, vg, vt, cache.k.data_ptr() + step,
                cache.v.data_ptr() + step, cache.num_pages, G, cache.page_size, cache.table.data_ptr(), cache.lengths.data_ptr(),
                at, S, cache.max_pages, T, nat.stream_of(device))


def page_truncate(cache: PagedCache, lengths=0) -> None:
    """Every slot shortened to at most `lengths` positions (an int, or int32 [slots] on the device, a tensor of its own; a
    negative one is 0): the pages past them are given back. Rows stay in memory, outside every read."""
    at, each = _per_slot(cache, lengths, "lengths")
    nat.call_on(cache.device, "attnlab_page_truncate", cache.table.data_ptr(), cache.lengths.data_ptr(), cache.refs.data_ptr(), at,
                each, cache.slots, cache.max_pages, cache.num_pages, cache.page_size, nat.stream_of(cache.device))


def page_compact(cache: PagedCache) -> None:
    """The pages in use moved to the pool's low end, in every layer: with n of them, the i-th at or past n goes to the i-th
    free one below n, and the table and refs follow. The pools past n then hold no sequence's rows."""
    scratch, nbytes = _scratch(cache)
    nat.call_on(cache.device, "attnlab_page_compact", cache.k.data_ptr(), cache.v.data_ptr(), cache.layers, cache.num_pages,
                cache.groups, cache.page_size, cache.table.data_ptr(), cache.lengths.data_ptr(), cache.refs.data_ptr(),
                cache.slots, cache.max_pages, scratch.data_ptr(), nbytes, nat.stream_of(cache.device))
