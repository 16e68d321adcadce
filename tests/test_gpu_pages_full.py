"""The paged cache on the GPU in pools that run out, against the list model (oracle/pages.py), exactly; and that a slot's rows outlive a
copy that could not be served."""
from __future__ import annotations

import random

import pytest
import torch

from attention_lab import page_append, page_compact, page_fork, page_reserve, page_truncate, shared_prefix_attention
from attention_lab.hip_attend import attend_paged
from test_gpu_pages import fresh, gen, ints, same, write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 5])
def test_rows_outlive_a_full_pool(gpu, T):
    """Two branches share a partly filled page, no page is free, both reserve; pages are freed, both go back, and read the old rows."""
    cache, model = fresh(gpu, 1, 2, 3, 2, 5, 16, 4)
    write(cache, model, gpu, 1, [37, 0, 32])                     # three pages and two: none is free
    page_fork(cache, ints([0, 0, 2], gpu))
    model.fork([0, 0, 2])
    q = torch.randn(2, 2, 2, 1, 128, generator=gen(5)).to(torch.bfloat16).to(gpu)
    read = lambda: shared_prefix_attention(q, cache.k[1], cache.v[1], cache.table[:2], cache.lengths[:2].clone())  # noqa: E731
    before = read()
    write(cache, model, gpu, 50, [T, T, 0])
    same(cache, model)
    assert int(cache.missing) == 1 and cache.lengths.tolist() == [37 + T, 37 + T, 32]
    for graph in (False, True):                                  # a claim reads as no page, in every read
        p = cache.table.clone()
        p[0, 2] = -1
        out = [shared_prefix_attention(q, cache.k[1], cache.v[1], t[:2], cache.lengths[:2].clone()) for t in (cache.table, p)]
        assert torch.equal(*out)
        out = [attend_paged(q[:, :, :, 0], cache.k[1], cache.v[1], t[:2], length=37 + T) for t in (cache.table, p)]
        assert torch.equal(*out)
    page_truncate(cache, ints([37, 37, 0], gpu))
    model.truncate([37, 37, 0])
    same(cache, model)
    assert torch.equal(read(), before)
    write(cache, model, gpu, 90, [T, T, 0])                      # with pages free, each has its own
    same(cache, model)
    assert int(cache.missing) == 1 and cache.table[0, 2] != cache.table[1, 2]


def steps(seed, model, no_compaction):
    """Rounds of: slots that end or go back, a few that the others branch from, steps of one or some positions."""
    rng = random.Random(seed)
    S, W, page = len(model.table), len(model.table[0]), model.page
    for _ in range(8):
        yield "truncate", [rng.choice([0, 0, n, max(n - 1, 0), rng.randint(0, n), min(n, page * W // 2)]) for n in model.lengths]
        few = [rng.randrange(S) for _ in range(max(1, S // 8))]
        yield "write", [rng.randint(1, 2 * page) if i in few or rng.random() < 0.1 else 0 for i in range(S)]
        yield "fork", [rng.choice([i, rng.choice(few), rng.choice(few), rng.choice(few), -1]) for i in range(S)]
        for _ in range(rng.randint(1, 3)):
            tokens = [rng.choice([0, 1, 1, 1, rng.randint(1, page + 1)]) for _ in range(S)]
            yield "write", tokens if any(tokens) else [1] * S
        if rng.random() < 0.5:
            yield "truncate", [rng.choice([n, n, n + 3, max(n - 1, 0), max(n - 3, 0), max(n - page, 0)]) for n in model.lengths]
            yield "write", [1] * S
        if not no_compaction and rng.random() < 0.5:
            yield "compact", None
        yield "fork", [rng.choice([i, i, rng.randrange(S)]) for i in range(S)]


@pytest.mark.parametrize("seed,S,G,page,W,pages", [
    (5, 3, 1, 4, 4, 5), (56, 5, 2, 8, 5, 9), (8, 9, 1, 2, 6, 13), (4, 33, 1, 16, 4, 30), (2, 4, 3, 64, 3, 5), (6, 300, 1, 4, 5, 400),
    (7, 1024, 1, 2, 4, 900), (3, 7, 1, 32, 6, 11), (3, 3, 1, 256, 3, 4), (10, 64, 2, 8, 6, 17000), (11, 6, 1, 8, 6, 40000),
])
def test_walk(gpu, seed, S, G, page, W, pages):
    """Random operations with hardly a page to spare (in the large pools most are taken by counts of no table's)."""
    cache, model = fresh(gpu, seed, 1, S, G, pages, page, W)
    free = min(pages, max(2, S * W // 4))
    held = pages - free
    if held > 1000:      # at the pool's end but for two pages, so that free ones lie in every round of the search
        cache.refs[2:2 + held] = 1
        taken = list(range(2, 2 + held))
    else:
        taken = []

    class Taken(type(model)):
        @property
        def refs(self):
            n = super().refs
            for p in taken:
                n[p] += 1
            return n

        def compact(self):
            pass

    model.__class__ = Taken
    claims = 0
    for op, arg in steps(seed, model, bool(taken)):
        if op == "write":
            write(cache, model, gpu, 100 * claims, arg)
        elif op == "fork":
            page_fork(cache, ints(arg, gpu))
            model.fork(arg)
        elif op == "truncate":
            page_truncate(cache, ints(arg, gpu))
            model.truncate(arg)
        else:
            page_compact(cache)
            super(Taken, model).compact()
        same(cache, model)
        claims += sum(entry < -1 for row in model.table for entry in row)
    assert claims > 0


def test_pinned_page_in_a_full_pool(gpu):
    """A page whose count is raised by hand is not written in place, though none is left for its holder."""
    cache, model = fresh(gpu, 6, 1, 1, 1, 2, 16, 4)
    write(cache, model, gpu, 1, [21])
    cache.refs[1] += 1
    kept = cache.k.clone()
    rows = torch.randn(1, 1, 4, 128, generator=gen(7)).to(torch.bfloat16).to(gpu)
    page_reserve(cache, 4)
    page_append(cache, 0, rows, rows)
    assert torch.equal(cache.k, kept) and cache.table[0].tolist() == [0, model.claim(1, 5), -1, -1]
    assert cache.refs.tolist() == [1, 2] and int(cache.missing) == 1
    page_truncate(cache, 21)
    assert cache.table[0].tolist() == [0, 1, -1, -1] and cache.refs.tolist() == [1, 2]


def test_in_a_graph(gpu):
    """A captured step in a pool that runs out and is relieved between replays."""
    cache, model = fresh(gpu, 8, 1, 4, 1, 7, 8, 6)
    write(cache, model, gpu, 1, [21, 0, 0, 0])
    tokens, parents, to = ints([1] * 4, gpu), ints([0] * 4, gpu), ints([99] * 4, gpu)
    k = torch.zeros(4, 1, 1, 128, dtype=torch.bfloat16, device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        page_truncate(cache, to)
        page_fork(cache, parents)
        page_reserve(cache, tokens)
        page_append(cache, 0, k, -k, tokens)
    rng = random.Random(3)
    for step in range(12):
        ps = [0] * 4 if step == 0 else [rng.choice([i, i, rng.randrange(4)]) for i in range(4)]
        ls = [99] * 4 if step % 3 else [rng.randint(0, n) for n in model.lengths]
        x = torch.randn(4, 1, 1, 128, generator=gen(step)).to(torch.bfloat16)
        for t, y in ((parents, ints(ps, gpu)), (to, ints(ls, gpu)), (k, x)):
            t.copy_(y)
        graph.replay()
        model.truncate(ls)
        model.fork(ps)
        model.reserve([1] * 4)
        model.append(0, x, -x, [1] * 4)
        same(cache, model)
        write(cache, model, gpu, 700 + step, [1, 0, 2, 0])       # eager work between replays
        same(cache, model)


def test_lengths_past_31_bits(gpu):
    """A slot that grows past 2^31 - 1 positions: no row of it is written any more, least of all over those it has."""
    cache, model = fresh(gpu, 9, 1, 2, 2, 8, 8, 4)
    write(cache, model, gpu, 1, [5, 3])
    tokens = [2 ** 31 - 1, 2]
    page_reserve(cache, ints(tokens, gpu))
    model.reserve([40, 2])                                       # as far as pages go, 40 positions are as many
    rows = torch.randn(2, 2, 2, 128, generator=gen(4)).to(torch.bfloat16)
    page_append(cache, 0, rows.to(gpu), rows.to(gpu), ints(tokens, gpu))
    model.append(0, rows, rows, [0, 2])
    assert cache.lengths.tolist() == [2 ** 31 - 1, 5] and cache.table.tolist() == model.table
    assert torch.equal(cache.k.cpu(), model.k) and torch.equal(cache.v.cpu(), model.v)
    page_truncate(cache, 5)
    model.truncate([5, 5])
    cache.missing.fill_(model.missing)
    same(cache, model)
