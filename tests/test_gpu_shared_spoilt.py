"""Keys and values that are not finite at positions that only some queries of the shared read see: those queries are spoilt, no other."""
from __future__ import annotations

import pytest
import torch

from test_gpu_shared import Case, make

pytestmark = pytest.mark.gpu
NAMES = ["one_run", "wide", "ragged_runs", "narrow_runs", "page_2", "no_runs", "chunk_2", "chunk_17", "chunk_130", "chunk_alone",
         "chunk_runs", "chunk_sixteen_heads"]


def put(c, x, b, j, value):
    """value into every dimension of position j of sequence b, K's or V's."""
    x[c.table[b][j // c.page], :, j % c.page] = value


def own(c, b):
    """The first position of sequence b's own pages."""
    for r, p in enumerate(c.prefixes):
        if c.runs[r] <= b < c.runs[r + 1]:
            return p // c.page * c.page
    return 0


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("parts", [None, (1, 3)])
def test_own_positions(gpu, name, bad, which, parts):
    """In the own part of some sequences, at the last position, in the chunk's middle, at its first one and before it."""
    clean = make(name, 5)
    want = clean.call(gpu, partitions=parts).float().cpu()
    n_seq = len(clean.lengths)
    for back in sorted({1, 2, (clean.T + 1) // 2, clean.T, clean.T + 1}):
        c = make(name, 5)
        hit = [b for b in range(0, n_seq, 3) if c.lengths[b] - back >= own(c, b)]
        for b in hit:
            put(c, getattr(c, which), b, c.lengths[b] - back, float(bad))
        got = c.call(gpu, partitions=parts).float().cpu()
        for b in range(n_seq):
            sees = [t for t in range(c.T) if b in hit and c.lengths[b] - back <= c.lengths[b] - c.T + t]
            blind = [t for t in range(c.T) if t not in sees]
            assert torch.isfinite(got[b][:, :, blind]).all(), (back, b)
            # the values of other queries are what they are without it, but for a second pass' order of sums and its rounding
            assert (got[b][:, :, blind] - want[b][:, :, blind]).abs().le(2.0 ** -7 * want[b][:, :, blind].abs() + 2.0 ** -7).all()
            if bad == "nan" or which == "v":   # an infinite key can weigh nothing
                assert not torch.isfinite(got[b][:, :, sees]).any(), (back, b)


@pytest.mark.parametrize("name", ["one_run", "wide", "ragged_runs", "narrow_runs", "chunk_17", "chunk_runs"])
@pytest.mark.parametrize("which", ["k", "v"])
def test_shared_positions(gpu, name, which):
    """In a run's shared pages: all of the run's sequences, and none of another's."""
    for at in (0, -1):
        c = make(name, 5)
        r = len(c.prefixes) - 1
        whole = c.prefixes[r] // c.page * c.page
        j = 0 if at == 0 else whole - 1
        put(c, getattr(c, which), c.runs[r], j, float("nan"))
        got = c.call(gpu).float()
        for b in range(len(c.lengths)):
            if c.runs[r] <= b < c.runs[r + 1]:
                assert not torch.isfinite(got[b]).any(), (at, b)
            else:
                assert torch.isfinite(got[b]).all(), (at, b)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_behind_the_sequence(gpu, T):
    """Rows of a sequence's pages past its length, which the next steps will write: nothing of them is read, whatever they hold."""
    for bad in (float("nan"), float("inf"), -3e38):
        c = Case(6, [5, 2], [64, 32], [64 + T + 1 + 7 * i for i in range(5)] + [90, 101], 16, 2, 3, T)
        want = c.call(gpu)
        for i, n in enumerate(c.lengths):
            for j in range(n, -(-n // c.page) * c.page):
                put(c, c.k, i, j, bad)
                put(c, c.v, i, j, bad)
        assert torch.equal(c.call(gpu), want)
