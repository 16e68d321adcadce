"""The shared read at the sizes where its shares and merges change rules: more tiles of rows than workgroups, in one round or several,
and rows of more partials than a half wave has lanes. Sampled rows against float64, with test_gpu_shared's bound (2^-16 in the place
of 2^-8 of a weight for one query)."""
from __future__ import annotations

import math
import random

import pytest
import torch

from attention_lab import shared_prefix_attention

pytestmark = pytest.mark.gpu
LOG2E = math.log2(math.e)


class Big:
    """Runs of sequences over shuffled pages; rows that nothing may read hold NaN."""

    def __init__(self, gpu, seed, sizes, prefixes, suffix, page, G, h, T):
        rng = random.Random(seed)
        g = torch.Generator(device=gpu).manual_seed(seed)
        self.T, self.G, self.h, self.page = T, G, h, page
        self.sizes, self.prefixes = sizes, prefixes
        self.lengths = [p + T - 1 + rng.randint(*suffix) for s, p in zip(sizes, prefixes) for _ in range(s)]
        B, W = len(self.lengths), -(-max(self.lengths) // page) + 1
        table, pages, b = torch.full((B, W), -1, dtype=torch.int64), 0, 0
        for s, p in zip(sizes, prefixes):
            common = p // page
            table[b:b + s, :common] = torch.arange(pages, pages + common)
            pages += common
            for i in range(b, b + s):
                own = -(-self.lengths[i] // page) - common
                table[i, common:common + own] = torch.arange(pages, pages + own)
                pages += own
            b += s
        perm = torch.randperm(pages + 2, generator=torch.Generator().manual_seed(seed))
        self.table = torch.where(table >= 0, perm[table.clamp(min=0)], -1).to(gpu)
        self.k, self.v = (torch.randn(pages + 2, G, page, 128, device=gpu, generator=g).to(torch.bfloat16) for _ in "kv")
        seen = torch.zeros(pages + 2, page, dtype=torch.bool, device=gpu)
        for i, n in enumerate(self.lengths):
            at = torch.arange(n, device=gpu)
            seen[self.table[i, at // page], at % page] = True
        for x in (self.k, self.v):
            x.masked_fill_(~seen[:, None, :, None], float("nan"))
        self.q = torch.randn(B, G, h, T, 128, device=gpu, generator=g).to(torch.bfloat16)
        self.rng, self.gpu = rng, gpu

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.gpu)

    def call(self, **kw):
        runs = [sum(self.sizes[:i]) for i in range(len(self.sizes) + 1)]
        return shared_prefix_attention(self.q, self.k, self.v, self.table.to(torch.int32), self.ints(self.lengths),
                                       self.ints(self.prefixes), runs=self.ints(runs), **kw)

    def tiles(self, rows):
        """Tiles of `rows` rows over all groups."""
        return self.G * sum(-(-s * self.T * self.h // rows) for s in self.sizes)

    def check(self, got, samples=24):
        assert torch.isfinite(got).all()
        B, weight = len(self.lengths), 2.0 ** -16 if self.T == 1 else 2.0 ** -8
        some = {(0, 0), (B - 1, self.T - 1), (0, self.T - 1), (B - 1, 0)}
        some |= {(self.rng.randrange(B), self.rng.randrange(self.T)) for _ in range(samples)}
        for b, t in sorted(some):
            at = torch.arange(self.lengths[b] - self.T + t + 1, device=self.gpu)
            k, v = (x[self.table[b, at // self.page], :, at % self.page].double().transpose(0, 1).contiguous() for x in (self.k, self.v))
            s = torch.matmul(k, self.q[b, :, :, t].double().transpose(1, 2).contiguous()) / 128 ** 0.5     # [G, keys, h]
            w = torch.softmax(s, dim=1).transpose(1, 2).contiguous()
            want, size = torch.matmul(w, v), torch.matmul(w, v.abs())
            err = 2.0 ** -8 * want.abs() + size * (weight + 2 * (2.0 ** -17 + (s.abs().max() * LOG2E + 8) * 2.0 ** -20))
            off = ((got[b, :, :, t].double() - want).abs() / err).max()
            assert off <= 1, (b, t, float(off))


@pytest.mark.parametrize("sizes,prefixes,suffix,page,G,h,partitions,least", [
    ([2], [12400], (1, 40), 16, 8, 4, None, 33),                 # narrow tiles, 48 shared partials
    ([4], [12400], (300, 900), 64, 8, 4, None, 33),              # wide ones, 32 and the own part's
    ([1], [9000], (1, 9), 16, 8, 3, None, 33),
    ([3], [20000], (4000, 4300), 64, 1, 2, (64, 64), 65),
    ([2], [17000], (16300, 16700), 64, 1, 4, (64, 64), 97),
    ([6, 6], [17000, 12000], (16300, 16700), 128, 1, 4, (64, 64), 97),
    ([3], [17000], (16300, 16700), 4, 1, 2, (64, 64), 97),
])
def test_many_partials(gpu, sizes, prefixes, suffix, page, G, h, partitions, least):
    c = Big(gpu, 1, sizes, prefixes, suffix, page, G, h, 1)
    if partitions:   # both parts in as many pieces of 256 keys as there is room for
        assert min(64, prefixes[0] // 256) + min(64, suffix[0] // 256) >= least
    c.check(c.call(partitions=partitions))


CHUNKS = [   # sizes, prefixes, suffix, page, h, T: tiles of 128 rows over 8 groups; 512 workgroups
    ([16], [1000], (1, 60), 64, 4, 140, 560),
    ([16], [6000], (1, 60), 64, 4, 140, 560),                    # 64 blocks and more: two rounds of even shares
    ([16], [5000], (1, 60), 64, 8, 150, 1200),                   # three
    ([9, 1, 7], [4200, 64, 7000], (1, 40), 32, 4, 150, 640),
    ([16], [4224], (1, 20), 64, 16, 256, 4096),                  # eight rounds and more: whole tiles
    ([5, 11], [130, 64], (1, 30), 8, 4, 140, 560),
]


@pytest.mark.parametrize("sizes,prefixes,suffix,page,h,T,tiles", CHUNKS)
def test_chunks_of_more_tiles_than_workgroups(gpu, sizes, prefixes, suffix, page, h, T, tiles):
    c = Big(gpu, 2, sizes, prefixes, suffix, page, 8, h, T)
    assert c.tiles(128) >= tiles > 512
    c.check(c.call(), samples=12)


@pytest.mark.parametrize("prefix", [(40, 300), (2100, 2300), (2048, 6000)])
@pytest.mark.parametrize("page", [4, 16])
def test_narrow_tiles_more_than_workgroups(gpu, prefix, page):
    """Runs of up to eight rows, over 768 tiles of sixteen: whole, and (64 tiles of 32 keys and more) even shares."""
    rng = random.Random(5)
    R = 100 if prefix[0] < 1000 else 110
    c = Big(gpu, 3, [1] * R, [rng.randint(*prefix) for _ in range(R)], (1, 30), page, 8, 8, 1)
    assert c.tiles(16) > 768
    c.check(c.call())


@pytest.mark.parametrize("sizes,prefixes,h", [([520], [1000], 8), ([520], [5000], 8), ([13] * 40, [4200 + 97 * i for i in range(40)], 8),
                                              ([300, 1, 230], [4500, 900, 100], 8), ([2100], [300], 16)])
def test_wide_tiles_more_than_workgroups(gpu, sizes, prefixes, h):
    """One query each, over 256 tiles of 128 rows."""
    c = Big(gpu, 4, sizes, prefixes, (1, 70), 64, 8, h, 1)
    assert c.tiles(128) > 256
    c.check(c.call())
