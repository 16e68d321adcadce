"""The paged cache on the GPU against the list model (oracle/pages.py): tables, lengths, counts and every row of the pools are
equal after every operation, exactly."""
from __future__ import annotations

import random

import pytest
import torch

from attention_lab import PagedCache, page_append, page_compact, page_fork, page_reserve, page_truncate
from attention_lab.hip_attend import attend_paged
from oracle.pages import Pages

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def fresh(gpu, seed, layers, S, G, pages, page, W):
    """An empty cache over pools of random rows, and its model."""
    k, v = (torch.randn(layers, pages, G, page, 128, generator=gen(seed + i)).to(torch.bfloat16) for i in (0, 1))
    cache = PagedCache.empty(layers, S, G, pages, page, W, device=gpu)
    cache.k.copy_(k)
    cache.v.copy_(v)
    return cache, Pages(k, v, cache.table.tolist(), cache.lengths.tolist())


def same(cache, model):
    assert cache.table.tolist() == model.table
    assert cache.lengths.tolist() == model.lengths
    assert cache.refs.tolist() == model.refs
    assert cache.missing.tolist() == [model.missing]
    assert torch.equal(cache.k.cpu(), model.k) and torch.equal(cache.v.cpu(), model.v)


def write(cache, model, gpu, seed, tokens, each=None):
    """Reserve and append in cache and model; `each`: the int form."""
    S, T = cache.slots, max(tokens)
    at = None if each else ints(tokens, gpu)
    page_reserve(cache, each if each else at)
    model.reserve(tokens)
    for layer in range(cache.layers):
        k, v = (torch.randn(S, T, cache.groups, 128, generator=gen(seed + 2 * layer + i)).to(torch.bfloat16).transpose(1, 2)
                for i in (0, 1))
        page_append(cache, layer, k.to(gpu), v.to(gpu), at)
        model.append(layer, k, v, tokens)


@pytest.mark.parametrize("seed,layers,S,G,pages,page,W", [
    (1, 2, 3, 2, 24, 4, 6), (2, 1, 1, 1, 5, 8, 5), (3, 1, 17, 3, 200, 1, 30), (4, 3, 9, 1, 40, 16, 5), (5, 1, 64, 2, 300, 2, 40),
    (6, 2, 5, 8, 33, 32, 4), (7, 1, 300, 1, 1500, 2, 9), (8, 1, 1024, 1, 3000, 1, 5), (9, 1, 4, 1, 20000, 1, 6001),
    (10, 1, 7, 2, 40, 64, 9),
])
def test_walk(gpu, seed, layers, S, G, pages, page, W):
    """Random operations, among them pages and table entries that run out and parents outside the slots."""
    cache, model = fresh(gpu, seed, layers, S, G, pages, page, W)
    rng = random.Random(seed)
    for step in range(25):
        op = rng.choice(["write", "write", "write", "fork", "truncate", "compact"]) if step else "write"
        if op == "write":
            most = rng.choice([1, 1, 2 * page + 1, W * page // 3 + 1])
            if rng.random() < 0.3:
                each = rng.randint(1, max(1, min(most, 40)))
                write(cache, model, gpu, 100 * step, [each] * S, each)
            else:
                tokens = [rng.choice([0, 1, rng.randint(1, most)]) for _ in range(S)]
                write(cache, model, gpu, 100 * step, tokens if any(tokens) else [1] * S)
        elif op == "fork":
            few = [rng.randrange(S) for _ in range(max(1, S // 3))]
            parents = [rng.choice([i, rng.choice(few), rng.choice(few), -1, S, rng.randrange(S)]) for i in range(S)]
            page_fork(cache, ints(parents, gpu))
            model.fork(parents)
        elif op == "truncate":
            to = [rng.choice([0, -1, n, n + 3, rng.randint(0, n), n - n % page, max(n - 1, 0)]) for n in model.lengths]
            page_truncate(cache, ints(to, gpu))
            model.truncate(to)
        else:
            page_compact(cache)
            model.compact()
            used = sum(r > 0 for r in model.refs)
            assert all(p < used for row in model.table for p in row)
        same(cache, model)


def test_beams(gpu):
    """A prompt, its branches, some steps of a beam search, a draft and its rollback, an end: what the sequences read back is
    what each was written, row by row."""
    cache, model = fresh(gpu, 11, 2, 6, 2, 64, 8, 12)
    write(cache, model, gpu, 1, [37, 0, 0, 0, 0, 0])
    page_fork(cache, ints([0] * 6, gpu))
    model.fork([0] * 6)
    assert cache.refs[:5].tolist() == [6] * 5                     # five pages held by all six
    for step, parents in enumerate(([0, 1, 2, 3, 4, 5], [0, 0, 2, 2, 5, 5], [5, 4, 3, 2, 1, 0], [1, 1, 1, 1, 1, 1])):
        page_fork(cache, ints(parents, gpu))
        model.fork(parents)
        write(cache, model, gpu, 50 + 10 * step, [1] * 6, 1)
        same(cache, model)
    write(cache, model, gpu, 200, [7] * 6)
    page_truncate(cache, 43)
    model.truncate([43] * 6)
    same(cache, model)
    page_truncate(cache, ints([0, 50, 0, 50, 0, 50], gpu))
    model.truncate([0, 50, 0, 50, 0, 50])
    page_compact(cache)
    model.compact()
    same(cache, model)
    for layer in range(2):
        q = torch.randn(6, 2, 2, 128, generator=gen(9 + layer)).to(torch.bfloat16).to(gpu)
        out = attend_paged(q, cache.k[layer], cache.v[layer], cache.table, length=43, out_dtype=torch.float32)
        for i in (1, 3, 5):
            k, v = (x.double() for x in model.rows(layer, i))
            s = q[i].double().cpu() @ k.transpose(1, 2) / 128 ** 0.5
            want = torch.softmax(s, dim=-1) @ v
            # fp32 sums of 128 products and 43 weighted rows, exp2 of a score below 16: 2^-17 of the largest value
            assert (out[i].double().cpu() - want).abs().max() <= 2.0 ** -17 * v.abs().max()


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 200])
@pytest.mark.parametrize("layout", ["rows", "heads", "odd", "repeated"])
def test_append_layouts(gpu, T, layout):
    """Strides, rows at odd addresses, tokens fewer than the rows, more slots than are written to."""
    cache, model = fresh(gpu, 3, 1, 4, 3, 64, 16, 16)
    tokens = [T, 0, max(T - 3, 0), min(T, 1)]
    page_reserve(cache, ints([5, 3, 16, 0], gpu))
    model.reserve([5, 3, 16, 0])
    page_reserve(cache, ints(tokens, gpu))
    model.reserve(tokens)
    made = []
    for i in (0, 1):
        if layout == "rows":
            x = torch.randn(4, 3, T, 128, generator=gen(T + i)).to(torch.bfloat16).to(gpu)
        elif layout == "heads":
            x = torch.randn(4, T, 3, 128, generator=gen(T + i)).to(torch.bfloat16).to(gpu).transpose(1, 2)
        elif layout == "odd":
            x = torch.randn(4 * 3 * T * 128 + 3, generator=gen(T + i)).to(torch.bfloat16).to(gpu)[3:].view(4, 3, T, 128)
        else:
            x = torch.randn(4, 1, 1, 128, generator=gen(T + i)).to(torch.bfloat16).to(gpu).expand(4, 3, T, 128)
        made.append(x)
    page_append(cache, 0, *made, ints(tokens, gpu))
    model.append(0, *(x.cpu() for x in made), tokens)
    same(cache, model)


def test_foreign_tables(gpu):
    """Entries that name no page, negative lengths and tokens: skipped, never followed."""
    cache, model = fresh(gpu, 5, 1, 4, 1, 16, 4, 6)
    table = [[0, 99, -7, -1, -1, -1], [16, 2, -1, -1, -1, -1], [-1] * 6, [2, 1, -1, -1, -1, -1]]
    cache.table.copy_(ints(table, gpu))
    cache.lengths.copy_(ints([9, 7, -5, 8], gpu))
    cache.refs.copy_(ints([1, 1, 2] + [0] * 13, gpu))
    model.table, model.lengths = [list(r) for r in table], [9, 7, 0, 8]
    tokens = [2, 1, -4, 1]
    page_reserve(cache, ints(tokens, gpu))
    model.reserve(tokens)
    model.lengths[2] = -5
    rows = torch.randn(4, 1, 2, 128, generator=gen(0)).to(torch.bfloat16)
    page_append(cache, 0, rows.to(gpu), rows.to(gpu), ints(tokens, gpu))
    model.append(0, rows, rows, tokens)
    same(cache, model)
    parents = [3, -2147483648, 2147483647, 0]
    page_fork(cache, ints(parents, gpu))
    model.fork(parents)
    assert cache.table.tolist() == model.table and cache.refs.tolist() == model.refs


def test_pinned_page(gpu):
    """A count raised by hand keeps a page from being written in place, in a cache of one slot too, and from being given out."""
    cache, model = fresh(gpu, 6, 2, 1, 2, 8, 16, 4)
    write(cache, model, gpu, 1, [21])
    kept = cache.k[:, 1].clone()
    cache.refs[1] += 1
    rows = torch.randn(2, 1, 2, 4, 128, generator=gen(7)).to(torch.bfloat16).to(gpu)
    page_reserve(cache, 4)
    for layer in range(2):
        page_append(cache, layer, rows[layer], rows[layer])
    assert cache.table[0, :2].tolist() == [0, 2] and cache.refs.tolist() == [1, 1, 1, 0, 0, 0, 0, 0]
    assert torch.equal(cache.k[:, 1], kept) and torch.equal(cache.k[:, 2, :, :5], kept[:, :, :5])
    assert torch.equal(cache.k[:, 2, :, 5:9], rows[:, 0])
    page_truncate(cache)
    assert cache.refs.tolist() == [0, 1, 0, 0, 0, 0, 0, 0]
    page_compact(cache)
    assert cache.refs.tolist() == [1, 0, 0, 0, 0, 0, 0, 0] and torch.equal(cache.k[:, 0], kept)


def test_step_in_a_graph(gpu):
    """Fork, reserve, append, truncate and compact captured once and replayed with other parents, tokens and rows, with eager
    work between: every replay equals the model."""
    cache, model = fresh(gpu, 21, 2, 5, 2, 60, 8, 12)
    write(cache, model, gpu, 1, [21, 9, 0, 3, 8])
    parents, tokens, to = ints([0, 1, 2, 3, 4], gpu), ints([1] * 5, gpu), ints([99] * 5, gpu)
    k, v = (torch.zeros(2, 5, 2, 3, 128, dtype=torch.bfloat16, device=gpu) for _ in "kv")
    before = [t.clone() for t in (cache.table, cache.lengths, cache.refs, cache.k, cache.v)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        page_fork(cache, parents)
        page_reserve(cache, tokens)
        for layer in range(2):
            page_append(cache, layer, k[layer], v[layer], tokens)
        page_truncate(cache, to)
        page_compact(cache)
    for t, b in zip((cache.table, cache.lengths, cache.refs, cache.k, cache.v), before):
        assert torch.equal(t, b)                                  # captured, not run
    rng = random.Random(2)
    for step in range(6):
        ps, ts = [rng.randrange(-1, 5) for _ in range(5)], [rng.randrange(0, 4) for _ in range(5)]
        ls = [rng.randrange(5, 40) for _ in range(5)]
        rows = [torch.randn(2, 5, 2, 3, 128, generator=gen(step + i)).to(torch.bfloat16) for i in (0, 1)]
        for t, x in ((parents, ints(ps, gpu)), (tokens, ints(ts, gpu)), (to, ints(ls, gpu)), (k, rows[0]), (v, rows[1])):
            t.copy_(x)
        graph.replay()
        model.fork(ps)
        model.reserve(ts)
        for layer in range(2):
            model.append(layer, rows[0][layer], rows[1][layer], ts)
        model.truncate(ls)
        model.compact()
        same(cache, model)
        write(cache, model, gpu, 900 + step, [1] * 5, 1)          # eager work between replays
        same(cache, model)


def test_two_caches_on_two_streams(gpu):
    caches = [fresh(gpu, 31 + i, 1, 33, 2, 600, 4, 30) for i in range(2)]
    streams = [torch.cuda.Stream(gpu) for _ in caches]
    torch.cuda.synchronize()
    for step in range(8):
        for i, ((cache, model), stream) in enumerate(zip(caches, streams)):
            with torch.cuda.stream(stream):
                write(cache, model, gpu, 10 * step + i, [1 + (step + j) % 5 for j in range(33)])
                parents = [(3 * j + step + i) % 33 for j in range(33)]
                page_fork(cache, ints(parents, gpu))
                model.fork(parents)
    torch.cuda.synchronize()
    for cache, model in caches:
        same(cache, model)


def test_large_offsets(gpu):
    """A pool past 4 GiB: rows in its last pages, written, copied for a branch and moved."""
    pages, page, G = 9000, 256, 8                                 # 4.7 GB each of K and V
    cache = PagedCache.empty(1, 2, G, pages, page, 8, device=gpu)
    cache.refs[:pages - 2] = 1                                    # held by nobody's table: only the last two are free
    tokens = ints([130, 0], gpu)
    rows = torch.randn(2, G, 130, 128, generator=gen(1)).to(torch.bfloat16).to(gpu)
    page_reserve(cache, tokens)
    page_append(cache, 0, rows, -rows, tokens)
    page_fork(cache, ints([0, 0], gpu))
    page_reserve(cache, 1)
    assert cache.table[:, 0].tolist() == [pages - 1, pages - 2]
    for i in (0, 1):
        p = int(cache.table[i, 0])
        assert torch.equal(cache.k[0, p, :, :130], rows[0]) and torch.equal(cache.v[0, p, :, :130], -rows[0])
    cache.refs[10:20] = 0
    page_compact(cache)
    assert sorted(cache.table[:, 0].tolist()) == [18, 19] and cache.table[0, 0] == 19
    for i in (0, 1):
        p = int(cache.table[i, 0])
        assert torch.equal(cache.k[0, p, :, :130], rows[0]) and torch.equal(cache.v[0, p, :, :130], -rows[0])
