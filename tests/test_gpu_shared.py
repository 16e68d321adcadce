"""Attention over shared prompts in a paged cache against float64, by each sequence's own table.

Per output element, with A = sum_j w_j |v_j| and S the largest |score| (log2): a weight is rounded to bf16, 2^-8, before the
product with V; its exponent is a product of fp32 sums over 128 exact products, at most (S + 8) 2^-20 relative to the weight, exp2
2^-22, sums over up to 2^17 rows in tiles and partials 2^-17, and weight and sum err alike (twice). The output is rounded once
more: 2^-8 of itself. Rows of the pools that no query may read hold NaN throughout.
"""
from __future__ import annotations

import math
import random
import threading

import pytest
import torch

from attention_lab import full_attention, shared_prefix_attention
from attention_lab.hip_attend import attend_paged

pytestmark = pytest.mark.gpu
LOG2E = math.log2(math.e)


def gen(seed):
    return torch.Generator().manual_seed(seed)


class Case:
    """Sequences in runs (sizes; a negative size: sequences of no run) with their tables, and pools that hold NaN elsewhere."""

    def __init__(self, seed, sizes, prefixes, lengths, page, G=2, h=2, T=1, spare=3):
        rng = random.Random(seed)
        self.T, self.page = T, page
        self.lengths = list(lengths)
        B = len(self.lengths)
        assert sum(abs(s) for s in sizes) == B
        W = max(1, -(-max(self.lengths + list(prefixes)) // page)) + 1
        self.table = [[-1] * W for _ in range(B)]
        pages = [0]

        def take():
            pages[0] += 1
            return pages[0] - 1

        self.runs, self.prefixes, b = [0] if sizes[0] > 0 else [-sizes[0]], [], 0
        given = iter(prefixes)
        for s in sizes:
            if s < 0:
                b -= s
                continue
            prefix = next(given)
            if self.runs[-1] != b:       # sequences of no run lie between: an empty prefix for them
                self.runs.append(b)
                self.prefixes.append(0)
            common = [take() for _ in range(prefix // page)]
            for i in range(b, b + s):
                self.table[i][:len(common)] = common
            b += s
            self.runs.append(b)
            self.prefixes.append(prefix)
        for i, n in enumerate(self.lengths):
            for e in range(-(-n // page)):
                if self.table[i][e] < 0:
                    self.table[i][e] = take()
        n = pages[0] + spare
        perm = list(range(n))
        rng.shuffle(perm)
        self.table = [[perm[p] if p >= 0 else p for p in row] for row in self.table]
        self.k, self.v = (torch.randn(n, G, page, 128, generator=gen(seed + i)).to(torch.bfloat16) for i in (0, 1))
        self.q = torch.randn(B, G, h, T, 128, generator=gen(seed + 2)).to(torch.bfloat16)
        self.unread()

    def legal(self, i):
        """(position, page, row) of the sequence's positions that have a page."""
        for j in range(min(self.lengths[i], len(self.table[i]) * self.page)):
            p = self.table[i][j // self.page]
            if 0 <= p < self.k.shape[0]:
                yield j, p, j % self.page

    def unread(self):
        seen = torch.zeros(self.k.shape[0], self.page, dtype=torch.bool)
        for i in range(len(self.lengths)):
            at = [(p, r) for _, p, r in self.legal(i)]
            if at:
                seen[tuple(torch.tensor(x) for x in zip(*at))] = True
        for x in (self.k, self.v):
            x.masked_fill_(~seen[:, None, :, None], float("nan"))

    def ints(self, gpu, x):
        return torch.tensor(x, dtype=torch.int32, device=gpu)

    def args(self, gpu):
        return (self.q.to(gpu), self.k.to(gpu), self.v.to(gpu), self.ints(gpu, self.table), self.ints(gpu, self.lengths),
                self.ints(gpu, self.prefixes) if self.prefixes else 0)

    def call(self, gpu, **kw):
        return shared_prefix_attention(*self.args(gpu), runs=self.ints(gpu, self.runs) if self.prefixes else None, **kw)

    def check(self, got, scale=None):
        sc = 128 ** -0.5 if scale is None else scale
        got = got.double().cpu()
        assert got.shape == self.q.shape
        for i, n in enumerate(self.lengths):
            n = min(n, len(self.table[i]) * self.page)
            at = list(self.legal(i))
            for t in range(self.T):
                seen = [(p, r) for j, p, r in at if j <= n - self.T + t]
                if not seen:
                    assert (got[i, :, :, t] == 0).all(), (i, t)
                    continue
                p, r = (torch.tensor(x) for x in zip(*seen))
                k, v = (x[p, :, r].double().transpose(0, 1) for x in (self.k, self.v))
                s = self.q[i, :, :, t].double() @ k.transpose(1, 2) * sc
                w = torch.softmax(s, dim=-1)
                want, size = w @ v, w @ v.abs()
                err = 2.0 ** -8 * want.abs() + size * (2.0 ** -8 + 2 * (2.0 ** -17 + (s.abs().max() * LOG2E + 8) * 2.0 ** -20))
                fine = torch.isfinite(want)
                assert torch.isfinite(got[i, :, :, t][fine]).all(), (i, t)
                assert not torch.isfinite(got[i, :, :, t][~fine]).any(), (i, t)
                assert ((got[i, :, :, t] - want).abs() <= err)[fine].all(), (i, t, ((got[i, :, :, t] - want).abs() / err).max())


def spread(rng, n, lo, hi):
    return [rng.randint(lo, hi) for _ in range(n)]


CASES = {   # sizes, prefixes, suffix range, page, G, h, T
    "one_run": ([5], [200], (1, 50), 16, 2, 2, 1),
    "one_sequence": ([1], [64], (1, 1), 64, 1, 1, 1),
    "wide": ([40], [333], (1, 130), 32, 2, 4, 1),
    "wide_tiles": ([70], [640], (1, 9), 64, 1, 6, 1),
    "ragged_runs": ([1, 17, 3, 30], [100, 900, 64, 257], (1, 70), 16, 2, 3, 1),
    "narrow_runs": ([2, 1, 3, 2], [100, 900, 64, 257], (1, 70), 8, 3, 4, 1),
    "sixteen_heads": ([2, 3], [130, 70], (1, 40), 16, 1, 16, 1),
    "odd_heads": ([9, 4], [515, 129], (3, 300), 128, 2, 5, 1),
    "page_1": ([6, 5], [77, 40], (1, 40), 1, 1, 2, 1),
    "page_2": ([20], [301], (1, 33), 2, 1, 7, 1),
    "page_4096": ([6, 20], [4096, 5000], (1, 90), 4096, 1, 2, 1),
    "none_shared": ([4, 3], [15, 5], (1, 600), 16, 2, 2, 1),
    "no_runs": ([-6], [], (0, 500), 16, 2, 8, 1),
    "outside": ([-2, 3, -1, 4, -3], [320, 90], (1, 60), 16, 2, 2, 1),
    "many_runs": ([1, 2, 1] * 30, [17 * (i % 5) + 16 for i in range(90)], (1, 9), 16, 1, 1, 1),
    "long_own": ([3], [64], (1500, 2500), 64, 1, 4, 1),
    "chunk_2": ([5], [200], (2, 50), 16, 2, 2, 2),
    "chunk_17": ([3, 5], [200, 96], (17, 80), 16, 2, 3, 17),
    "chunk_130": ([4], [500], (130, 260), 64, 1, 2, 130),
    "chunk_alone": ([-3], [], (100, 100), 32, 2, 4, 100),
    "chunk_sixteen_heads": ([2], [70], (33, 40), 16, 1, 16, 33),
    "chunk_runs": ([2, 3, 1], [64, 640, 128], (65, 300), 128, 1, 1, 65),
    "chunk_one_row": ([2, 1], [64, 32], (3, 9), 16, 1, 1, 3),
}


def make(name, seed=1):
    sizes, prefixes, (lo, hi), page, G, h, T = CASES[name]
    rng = random.Random(seed)
    lengths, given = [], iter(prefixes)
    for s in sizes:
        base = next(given) if s > 0 else 0
        lengths += [base + rng.randint(lo, hi) for _ in range(abs(s))]
    return Case(seed, sizes, prefixes, lengths, page, G, h, T)


@pytest.mark.parametrize("name", list(CASES))
def test_cases(gpu, name):
    c = make(name)
    c.check(c.call(gpu))


@pytest.mark.parametrize("name", ["wide", "ragged_runs", "narrow_runs", "outside", "chunk_17", "chunk_130", "no_runs"])
@pytest.mark.parametrize("parts", [(0, 1), (1, 1), (2, 1), (3, 2), (64, 64), (0, 5)])
def test_partitions(gpu, name, parts):
    c = make(name, 2)
    c.check(c.call(gpu, partitions=parts))


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("sizes", [[12], [3, 1, 4, 4]])
def test_short_sequences(gpu, T, sizes):
    """Sequences that end inside their prefix, have no position, or fewer than queries; odd prefixes round down to pages."""
    rng = random.Random(T)
    for page in (8, 64):
        prefixes = [rng.randint(100, 300) for _ in sizes]
        lengths = []
        for s, p in zip(sizes, prefixes):
            lengths += [rng.choice([0, 1, T, p // 2, p - 1, p, p + T - 1, p + T, p + 37]) for _ in range(s)]
        for h in (1, 3):
            c = Case(T, sizes, prefixes, lengths, page, 1, h, T)
            c.check(c.call(gpu))


@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("n", [4, 70])
def test_ended_sequences(gpu, T, n):
    """Slots of a run whose sequences have ended, the first ones among them: empty tables, and the others read on."""
    lengths = [200 + i % 13 for i in range(n)]
    for alive in (range(1, n), range(n // 2, n), [n - 1], []):
        c = Case(12, [n, 3], [160, 64], lengths + [90, 91, 92], 16, 1, 2, T)
        for i in range(n):
            if i not in alive:
                c.table[i] = [-1] * len(c.table[i])
                c.lengths[i] = 0
        c.unread()
        c.check(c.call(gpu))


@pytest.mark.parametrize("T", [1, 40])
def test_missing_pages(gpu, T):
    """Entries that name no page, in the prefix and behind it, at the ends and all of them."""
    c = Case(4, [6, 20], [300, 128], [300 + 40 + 7 * i for i in range(6)] + [128 + 41 + i for i in range(20)], 16, 1, 2, T)
    pages = c.k.shape[0]
    for b in range(6):
        c.table[b][0], c.table[b][7] = -1, pages
    for b in range(6, 26):
        c.table[b][3:8] = [-5, 2 ** 31 - 1, -2 ** 31, -1, -1]
    c.table[2][18:] = [-1] * len(c.table[2][18:])
    c.table[9][8:] = [-1] * len(c.table[9][8:])
    c.unread()
    c.check(c.call(gpu))
    for row in c.table:
        row[:] = [-1] * len(row)
    c.check(c.call(gpu))


@pytest.mark.parametrize("name", ["wide", "narrow_runs", "chunk_17"])
@pytest.mark.parametrize("scale", [0.0, -0.09, 1e-40, 3.0])
def test_scales(gpu, name, scale):
    c = make(name, 3)
    c.check(c.call(gpu, scale=scale), scale)


@pytest.mark.parametrize("name,h", [("one_run", 2), ("wide", 4), ("chunk_17", 3), ("chunk_130", 2)])
def test_not_finite(gpu, name, h):
    """NaN and infinities in rows that some queries see and others do not: a query that sees them is spoilt, no other."""
    for bad in (float("nan"), float("inf")):
        c = make(name, 5)
        B = len(c.lengths)
        for b in range(0, B, 3):                     # the last position of some sequences
            j = c.lengths[b] - 1
            c.v[c.table[b][j // c.page], :, j % c.page, 5] = bad
        got = c.call(gpu).double().cpu()
        for b in range(B):
            for t in range(c.T):
                spoilt = b % 3 == 0 and t == c.T - 1
                assert torch.isfinite(got[b, :, :, t, 5]).all() == (not spoilt), (b, t)
                assert torch.isfinite(got[b, :, :, t, 6]).all()
        c = make(name, 5)
        c.k[c.table[1][c.lengths[1] // 2 // c.page], :, c.lengths[1] // 2 % c.page, 3] = float("nan")
        got = c.call(gpu).double().cpu()
        if c.lengths[1] // 2 >= c.prefixes[0] // c.page * c.page:
            assert torch.isfinite(got[0]).all()
        assert not torch.isfinite(got[1, :, :, -1]).any()


def test_loud_values(gpu):
    """Values near the type's end: weights are at most 1, sums stay finite."""
    for name in ("wide", "one_run", "chunk_17"):
        c = make(name, 6)
        c.v *= 2.0 ** 115
        got = c.call(gpu).float()
        assert torch.isfinite(got).all()
        c.check(got)


def test_layouts(gpu):
    """Queries of other strides and at odd addresses, a wider table's columns, one length and prefix for all, a given output."""
    c = make("one_run", 7)
    want = c.call(gpu)
    q, k, v, table, lengths, prefix = c.args(gpu)
    runs = c.ints(gpu, c.runs)
    turned = q.permute(4, 3, 2, 1, 0).contiguous().permute(4, 3, 2, 1, 0)
    assert torch.equal(shared_prefix_attention(turned, k, v, table, lengths, prefix, runs=runs), want)
    odd = torch.empty(q.numel() + 3, dtype=q.dtype, device=gpu)[3:].view(q.shape).copy_(q)
    assert torch.equal(shared_prefix_attention(odd, k, v, table, lengths, prefix, runs=runs), want)
    broad = torch.full((table.shape[0], table.shape[1] + 5), -1, dtype=torch.int32, device=gpu)
    broad[:, 2:2 + table.shape[1]] = table
    assert torch.equal(shared_prefix_attention(q, k, v, broad[:, 2:2 + table.shape[1]], lengths, prefix, runs=runs), want)
    assert torch.equal(shared_prefix_attention(q, k, v, table, lengths, c.prefixes[0]), want)
    out = torch.empty_like(q)
    assert shared_prefix_attention(q, k, v, table, lengths, prefix, runs=runs, out=out) is out and torch.equal(out, want)
    c.lengths = [210] * 5
    c = Case(7, [5], [200], c.lengths, 16)
    q, k, v, table, lengths, prefix = c.args(gpu)
    c.check(shared_prefix_attention(q, k, v, table, 210, 200))
    c.check(shared_prefix_attention(q, k, v, table, 210, prefix))
    assert shared_prefix_attention(q[:, :, :, :0], k, v, table, 210, 200).shape == (5, 2, 2, 0, 128)
    one = shared_prefix_attention(q[:1], k, v, table[:1], 210, 200)
    assert torch.allclose(one.float(), shared_prefix_attention(q, k, v, table, 210, 200)[:1].float(), atol=2e-2)


def test_beside_the_other_reads(gpu):
    """The paged read at one length, and the full read of the same rows in a contiguous cache."""
    for T in (1, 33):
        c = Case(8, [6], [256], [400] * 6, 16, 2, 4, T)
        got = c.call(gpu).double()
        c.check(got)
        q, k, v, table, *_ = c.args(gpu)
        if T == 1:
            other = attend_paged(q[:, :, :, 0].contiguous(), k, v, table, length=400, out_dtype=torch.float32)[:, :, :, None]
        else:
            rows = lambda x: x[table[:, :25].long()].transpose(1, 2).reshape(6, 2, 400, 128).contiguous()  # noqa: E731
            other = full_attention(q, rows(k), rows(v))
        c.check(other)


@pytest.mark.parametrize("runs", [[0, 9, 4, 12], [-3, 5, 2 ** 31 - 1, 7], [12, 0, 0, 5], [3, 3, 3, 3], [0, -1, -1, 100]])
def test_odd_runs(gpu, runs):
    """Bounds out of order and outside the batch: a run begins no earlier than the largest bound before it. The tables here
    agree everywhere, so any cut of the batch gives the same."""
    c = Case(9, [12], [128], [140 + i for i in range(12)], 16, 1, 2, 1)
    q, k, v, table, lengths, _ = c.args(gpu)
    c.check(shared_prefix_attention(q, k, v, table, lengths, c.ints(gpu, [128, 100, 128]), runs=c.ints(gpu, runs)))
    c.check(shared_prefix_attention(q, k, v, table, c.ints(gpu, [n for n in c.lengths]), 128, runs=c.ints(gpu, runs)))


def test_past_the_table(gpu):
    """Lengths and prefixes past what the table holds, and negative ones."""
    c = Case(10, [4], [96], [150, 160, 130, 100], 16, 1, 2, 1)
    q, k, v, table, lengths, _ = c.args(gpu)
    table = table[:, :9].contiguous()
    c.table = [row[:9] for row in c.table]
    c.lengths = [144, 144, 130, 100]
    c.unread()
    q, k, v, *_ = c.args(gpu)
    c.check(shared_prefix_attention(q, k, v, table, lengths, 96))
    c.check(shared_prefix_attention(q, k, v, table, c.ints(gpu, [2 ** 31 - 1, 145, 130, 100]), 96))
    c.check(shared_prefix_attention(q, k, v, table, lengths, c.ints(gpu, [-4])))
    c.lengths = [0, 144, 130, 0]
    c.check(shared_prefix_attention(q, k, v, table, c.ints(gpu, [-7, 160, 130, 0]), 96))


def test_graph(gpu):
    """One graph replayed over later lengths, prefixes, runs and rows, another one and eager calls between."""
    c = Case(11, [7, 9], [320, 160], [330 + i for i in range(7)] + [170 + 9 * i for i in range(9)], 16, 2, 2, 1)
    state = [*c.args(gpu), c.ints(gpu, c.runs)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(shared_prefix_attention(*state[:6], runs=state[6]))
        graphs.append(graph)
    for step in range(5):
        d = Case(20 + step, [7, 9], [320, 160], [330 + (i * step) % 15 for i in range(7)] + [170 + (7 * i + step) % 80 for i in range(9)],
                 16, 2, 2, 1)
        if step % 2:
            d.runs = [0, 5, 16] if step == 1 else [2, 7, 12]      # a cut inside a run shares as much
            d.prefixes = [300, 150] if step == 3 else [160, 0]
        n = d.k.shape[0]
        assert n <= state[1].shape[0] + 40
        for t, x in zip(state, [d.q, None, None, None, torch.tensor(d.lengths), torch.tensor(d.prefixes), torch.tensor(d.runs)]):
            if x is not None:
                t.copy_(x)
        pool = min(n, state[1].shape[0])
        keep = [[p if p < pool else -1 for p in row] for row in d.table]
        width = state[3].shape[1]
        d.table = [(row + [-1] * width)[:width] for row in keep]
        d.k, d.v = d.k[:pool], d.v[:pool]
        state[1][:pool].copy_(d.k)
        state[2][:pool].copy_(d.v)
        state[3].copy_(torch.tensor(d.table))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            d.check(out)
        assert torch.equal(shared_prefix_attention(*state[:6], runs=state[6]), outs[0])


def test_streams_and_threads(gpu):
    cases = [make("ragged_runs", 30), make("wide", 31)]
    want = [c.call(gpu) for c in cases]
    args = [(c.args(gpu), c.ints(gpu, c.runs)) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(gpu)):
            got[i] = [shared_prefix_attention(*args[i][0], runs=args[i][1]) for _ in range(20)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for w, many in zip(want, got):
        assert len(many) == 20 and all(torch.equal(w, x) for x in many)


def test_large_offsets(gpu):
    """Pools past 4 GiB: pages at their far end."""
    page, G = 256, 8
    for T in (1, 20):
        c = Case(40, [5], [512], [560, 600, 700, 541, 533], page, G, 2, T, spare=0)
        used, far = c.k.shape[0], 9000
        pools = [torch.full((far, G, page, 128), float("nan"), dtype=torch.bfloat16, device=gpu) for _ in "kv"]
        for pool, x in zip(pools, (c.k, c.v)):
            pool[far - used:].copy_(x)
        q, _, _, table, lengths, prefix = c.args(gpu)
        table = torch.where(table >= 0, table + far - used, table)
        c.check(shared_prefix_attention(q, *pools, table, lengths, prefix))
