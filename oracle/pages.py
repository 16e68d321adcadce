"""A paged K/V cache as lists and CPU tensors, one slot and one page at a time (no reference code). Test infrastructure only.

Pinned by known answers in tests/test_pages_host.py."""
from __future__ import annotations

import torch


class Pages:
    """k, v [layers, pages, G, page, d] CPU tensors; table, lengths and refs as lists."""

    def __init__(self, k, v, table, lengths, missing: int = 0):
        self.k, self.v = k.clone(), v.clone()
        self.table, self.lengths = [list(r) for r in table], list(lengths)
        self.pages, self.page = int(k.shape[1]), int(k.shape[3])
        self.missing = missing

    def claim(self, page, rows):
        """The entry of a slot that has the first `rows` rows of the page, and a length past them."""
        return -2 ** 31 + rows * self.pages + page

    def claimed(self, entry):
        """(page, rows) of such an entry; (-1, 0) of others."""
        rows, page = divmod(entry + 2 ** 31, self.pages)
        return (page, rows) if entry < -1 and 1 <= rows < self.page else (-1, 0)

    @property
    def refs(self):
        n = [0] * self.pages
        for row in self.table:
            for entry in row:
                p = self.claimed(entry)[0] if entry < 0 else entry
                if 0 <= p < self.pages:
                    n[p] += 1
        return n

    def fork(self, parents):
        S, W = len(self.table), len(self.table[0])
        ok = [0 <= p < S for p in parents]
        self.table = [list(self.table[p]) if o else [-1] * W for p, o in zip(parents, ok)]
        self.lengths = [self.lengths[p] if o else 0 for p, o in zip(parents, ok)]

    def truncate(self, to):
        for i, l in enumerate(to):
            n, l = self.lengths[i], max(l, 0)
            if l < n:
                self.lengths[i] = l
                for e in range(-(-l // self.page), len(self.table[i])):
                    self.table[i][e] = -1
                if l % self.page and l // self.page < len(self.table[i]):
                    page, rows = self.claimed(self.table[i][l // self.page])
                    if l % self.page <= rows:
                        self.table[i][l // self.page] = page

    def reserve(self, tokens):
        page, W = self.page, len(self.table[0])
        refs = self.refs
        grows = [(i, self.lengths[i], t) for i, t in enumerate(tokens) if t > 0]
        ends_in = {}
        for i, n, _ in grows:
            if n % page and n // page < W and 0 <= self.table[i][n // page] < self.pages:
                ends_in.setdefault(self.table[i][n // page], []).append(i)
        # all of the page's holders grow: the last keeps it
        away = {i for p, who in ends_in.items() for i in (who[:-1] if len(who) == refs[p] else who)}
        free = [p for p in range(self.pages) if refs[p] == 0]
        was, left = [list(row) for row in self.table], set()
        for i, n, t in grows:
            entries = ([n // page] if i in away else []) + list(range(-(-n // page), -(-(n + t) // page)))
            for e in entries:
                if e >= W:
                    self.missing += 1
                    continue
                p = free.pop(0) if free else -1
                if p < 0 and e < -(-n // page):
                    left.add(i)
                    continue
                self.missing += p < 0
                if e < -(-n // page):
                    for x in (self.k, self.v):
                        x[:, p, :, :n % page] = x[:, self.table[i][e], :, :n % page]
                self.table[i][e] = p
            self.lengths[i] = n + t
        # no page for a copy: the longest writer that is left writes on in place if the others claim no more, and those claim theirs
        part = {i: n % page for i, n, _ in grows}
        for p, who in ends_in.items():
            here = [i for i in who if i in left or i not in away]
            if not left & set(here):
                continue
            e = {i: n // page for i, n, _ in grows}[here[0]]
            claims = [self.claimed(row[e])[1] for row in was if self.claimed(row[e])[0] == p]
            best = max(here, key=lambda i: (part[i], i))
            on = len(who) + len(claims) == refs[p] and max(claims, default=0) <= part[best]
            for i in here:
                if not (on and i == best):
                    self.table[i][e] = self.claim(p, part[i])
                    self.missing += 1

    def append(self, layer, k, v, tokens):
        """k, v [S, G, T, d]."""
        for i, t in enumerate(tokens):
            for u in range(min(t, k.shape[2])):
                pos = self.lengths[i] - t + u
                e = pos // self.page
                p = self.table[i][e] if 0 <= e < len(self.table[i]) else -1
                if 0 <= p < self.pages:
                    self.k[layer, p, :, pos % self.page] = k[i, :, u]
                    self.v[layer, p, :, pos % self.page] = v[i, :, u]

    def compact(self):
        refs = self.refs
        used = [p for p in range(self.pages) if refs[p]]
        n = len(used)
        holes = [p for p in range(n) if not refs[p]]
        to = dict(zip([p for p in used if p >= n], holes))
        for src, dst in to.items():
            self.k[:, dst], self.v[:, dst] = self.k[:, src], self.v[:, src]
        def moved(entry):
            page, rows = self.claimed(entry)
            return self.claim(to[page], rows) if page in to else to.get(entry, entry)

        self.table = [[moved(entry) for entry in row] for row in self.table]

    def rows(self, layer, slot):
        """The slot's rows by position: (k, v) [G, length, d]; only where every position has a page."""
        pos = torch.arange(self.lengths[slot])
        at = torch.tensor(self.table[slot])[pos // self.page]
        return tuple(x[layer][at, :, pos % self.page].transpose(0, 1) for x in (self.k, self.v))
