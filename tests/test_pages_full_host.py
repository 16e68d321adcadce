"""The paged cache's model (oracle/pages.py) in pools that run out: known answers, and that no written row is ever lost or changed
for a slot that still has it."""
from __future__ import annotations

import random

import pytest
import torch

from oracle.pages import Pages


def model(S, pages, W, page):
    k = torch.zeros(1, pages, 1, page, 1, dtype=torch.float64)
    return Pages(k, k, [[-1] * W for _ in range(S)], [0] * S)


def claim(m, page, rows):
    return -2 ** 31 + rows * m.pages + page


def test_one_writes_on_the_other_claims():
    m = model(3, 3, 3, 4)
    m.reserve([6, 0, 4])                       # pages 0, 1 and 2: none is free
    m.fork([0, 0, 2])
    m.reserve([1, 1, 0])                       # all of page 1's holders grow: slot 1 keeps it, slot 0's copy is missing
    assert m.table == [[0, claim(m, 1, 2), -1], [0, 1, -1], [2, -1, -1]] and m.lengths == [7, 7, 4]
    assert m.refs == [2, 2, 1] and m.missing == 1
    m.reserve([0, 1, 0])                       # slot 0 claims two rows, slot 1 has three: in place again
    assert m.table[1] == [0, 1, -1] and m.missing == 1
    m.truncate([7, 9, 0])                      # nothing shorter than it was, but for slot 2
    assert m.table[0] == [0, claim(m, 1, 2), -1] and m.refs == [2, 2, 0]
    m.fork([0, 1, 0])
    assert m.table[2] == [0, claim(m, 1, 2), -1] and m.refs == [3, 3, 0]
    m.truncate([6, 9, 5])                      # back to where the rows end, or before
    assert m.table == [[0, 1, -1], [0, 1, -1], [0, 1, -1]] and m.lengths == [6, 8, 5] and m.refs == [3, 3, 0]
    m.reserve([1, 0, 0])
    assert m.table[0] == [0, 2, -1] and m.refs == [3, 2, 1] and m.missing == 1
    m.truncate([4, 0, 0])
    assert m.refs == [1, 0, 0] and m.table[0] == [0, -1, -1]


def test_a_claim_is_given_back():
    m = model(2, 2, 2, 4)
    m.reserve([6, 0])
    m.fork([0, 0])
    m.reserve([1, 1])
    assert m.table == [[0, claim(m, 1, 2)], [0, 1]]
    m.truncate([4, 9])
    assert m.table == [[0, -1], [0, 1]] and m.refs == [2, 1]


def test_shorter_writers_claim():
    """Of two writers in a full pool the longer one goes on, although the other is the last."""
    m = model(2, 2, 2, 8)
    m.reserve([14, 0])
    m.fork([0, 0])
    m.truncate([14, 11])
    m.reserve([1, 1])
    assert m.table == [[0, 1], [0, claim(m, 1, 3)]] and m.missing == 1 and m.refs == [2, 2]
    m.truncate([9, 11])                        # now the one in the page is the shorter one
    m.truncate([9, 99])
    m.reserve([2, 0])
    assert m.table[0] == [0, claim(m, 1, 1)] and m.refs == [2, 2] and m.missing == 2


def test_nobody_writes_on_beside_a_holder_that_does_not():
    m = model(3, 2, 2, 4)
    m.reserve([6, 0, 0])
    m.fork([0, 0, 0])
    m.reserve([0, 1, 1])
    assert m.table == [[0, 1]] + [[0, claim(m, 1, 2)]] * 2 and m.missing == 2 and m.refs == [3, 3]


def test_claims_move():
    m = model(2, 4, 2, 4)
    m.table, m.lengths = [[3, claim(m, 2, 1)], [0, 2]], [6, 7]
    assert m.refs == [1, 0, 2, 1]
    m.compact()
    assert m.refs == [1, 2, 1, 0] or m.refs == [1, 1, 2, 0]
    to = m.table[1][1]
    assert m.table == [[3 - to, claim(m, to, 1)], [0, to]] and m.refs[to] == 2


class Written:
    """What every position of every slot was written, beside a model."""

    def __init__(self, m):
        self.m, self.rows, self.next = m, [[] for _ in m.table], 1.0

    def write(self, tokens):
        m = self.m
        m.reserve(tokens)
        T = max([t for t in tokens if t > 0], default=0)
        x = torch.arange(len(tokens) * T, dtype=torch.float64).view(len(tokens), 1, T, 1) + self.next
        self.next += x.numel()
        m.append(0, x, -x, tokens)
        for i, t in enumerate(tokens):
            for u in range(max(t, 0)):
                e = len(self.rows[i]) // m.page
                there = e < len(m.table[i]) and m.table[i][e] >= 0
                self.rows[i].append(float(x[i, 0, u, 0]) if there else None)

    def fork(self, parents):
        self.m.fork(parents)
        self.rows = [list(self.rows[p]) if 0 <= p < len(self.rows) else [] for p in parents]

    def truncate(self, to):
        self.m.truncate(to)
        self.rows = [r[:max(n, 0)] for r, n in zip(self.rows, to)]

    def check(self):
        m = self.m
        for i, rows in enumerate(self.rows):
            assert m.lengths[i] == len(rows)
            for j, x in enumerate(rows):
                if x is None:
                    continue
                entry, r = m.table[i][j // m.page], j % m.page
                page, claimed = (entry, m.page) if entry >= 0 else m.claimed(entry)
                assert r < claimed, (i, j, entry)
                assert float(m.k[0, page, 0, r, 0]) == x and float(m.v[0, page, 0, r, 0]) == -x, (i, j, entry)
            # a whole row of positions without a page ends where a truncation makes all of them readable
            first = next((j for j, x in enumerate(rows) if x is None), len(rows))
            assert all(x is None for x in rows[first:-(-first // m.page) * m.page])


@pytest.mark.parametrize("seed", range(60))
def test_no_row_is_lost(seed):
    """Random operations in pools that are too small: every row that a slot was written stays its own, readable or claimed."""
    rng = random.Random(seed)
    S, page = rng.randint(2, 9), rng.choice([2, 4, 8, 16])
    W = rng.randint(2, 6)
    w = Written(model(S, rng.randint(2, max(3, S * W // 3)), W, page))
    for _ in range(120):
        op = rng.choice(["write"] * 4 + ["fork", "truncate", "truncate", "compact"])
        if op == "write":
            w.write([rng.choice([0, 1, 1, rng.randint(1, page + 2)]) for _ in range(S)] if rng.random() < 0.5 else [1] * S)
        elif op == "fork":
            few = [rng.randrange(S) for _ in range(2)]
            w.fork([rng.choice([i, i, rng.choice(few), rng.choice(few), -1]) for i in range(S)])
        elif op == "truncate":
            w.truncate([rng.choice([n, n, n + 2, max(n - 1, 0), rng.randint(0, n), next(
                (j for j, x in enumerate(w.rows[i]) if x is None), n)]) for i, n in enumerate(w.m.lengths)])
        else:
            w.m.compact()
        w.check()
        if rng.random() < 0.1:
            w.truncate([len(r) if rng.random() < 0.5 else 0 for r in w.rows])
