"""Page tables and the moves of a paged cache on the CPU, one sequence and one page after another, from their
description in include/bq.h. Written apart from the kernels; used by the tests alone."""
from __future__ import annotations


class Tables:
    """table: a list of lists of page numbers (-1 past the last), lens, refs: lists of ints."""

    def __init__(self, table, lens, refs, page):
        self.table, self.lens, self.refs, self.page = [list(r) for r in table], list(lens), list(refs), page

    def need(self, tokens):
        return (tokens + self.page - 1) // self.page if tokens > 0 else 0

    def cut(self, to):
        for s, row in enumerate(self.table):
            self.lens[s] = min(self.lens[s], max(to[s], 0))
            for c in range(self.need(self.lens[s]), len(row)):
                if row[c] >= 0:
                    if row[c] < len(self.refs):
                        self.refs[row[c]] -= 1
                    row[c] = -1

    def fork(self, parents):
        n, width = len(self.table), len(self.table[0]) if self.table else 0
        old, lens = [list(r) for r in self.table], list(self.lens)
        for s, p in enumerate(parents):
            real = 0 <= p < n
            self.table[s], self.lens[s] = (list(old[p]), lens[p]) if real else ([-1] * width, 0)
        for rows, by in ((old, -1), (self.table, 1)):
            for row in rows:
                for page in row:
                    if 0 <= page < len(self.refs):
                        self.refs[page] += by

    def last(self, s):
        """The page that sequence s would write to, partly filled, or None."""
        i, off = divmod(self.lens[s], self.page)
        if off == 0 or i >= len(self.table[s]):
            return None
        page = self.table[s][i]
        return page if 0 <= page < len(self.refs) else None

    def grow(self, more, rows):
        """cu, slots, at, moves, ok."""
        n, width = len(self.table), len(self.table[0]) if self.table else 0
        none = ([0] * (n + 1), [-1] * rows, [-1] * rows, [[-1] * n, [-1] * n, [0] * n], 0)
        if any(m < 0 or x < 0 or self.need(x + m) > width for m, x in zip(more, self.lens)) or sum(more) > rows:
            return none
        shared = {}
        for s in range(n):
            page = self.last(s)
            if more[s] > 0 and page is not None and self.refs[page] > 1:
                shared.setdefault(page, []).append(s)
        own = {s for page, who in shared.items() for s in (who[1:] if len(who) == self.refs[page] else who)}
        free = [p for p, r in enumerate(self.refs) if r == 0]
        wanted = sum(self.need(self.lens[s] + more[s]) - self.need(self.lens[s]) + (s in own) for s in range(n))
        if wanted > len(free):
            return none
        moves, cu, slots, at = [[-1] * n, [-1] * n, [0] * n], [0], [], []
        for s in range(n):
            if s in own:
                i, off = divmod(self.lens[s], self.page)
                src, dst = self.table[s][i], free.pop(0)
                self.refs[src] -= 1
                self.refs[dst] = 1
                self.table[s][i] = dst
                moves[0][s], moves[1][s], moves[2][s] = src, dst, off
            for c in range(self.need(self.lens[s]), self.need(self.lens[s] + more[s])):
                self.table[s][c] = free.pop(0)
                self.refs[self.table[s][c]] = 1
            for t in range(self.lens[s], self.lens[s] + more[s]):
                page = self.table[s][t // self.page]
                at.append(t)
                slots.append(page * self.page + t % self.page if 0 <= page < len(self.refs) else -1)
            self.lens[s] += more[s]
            cu.append(cu[-1] + more[s])
        blank = [-1] * (rows - len(at))
        return cu, slots + blank, at + blank, moves, 1
