"""Restatement of the page operators of include/kvpage.h on host arrays, one
row and one token at a time: the definition that the device kernels are
compared with."""
from __future__ import annotations

import numpy as np

ERR_PAGE, ERR_ROW, ERR_REFS, ERR_KEEP = 1, 2, 4, 8
OK, NO_PAGES, INVALID = 0, 1, 2


class Pages:
    """table [rows, width], lens [rows], refs [pages], the free stack, and a
    cache [planes, pages, block, unit bytes] (token-major)."""

    def __init__(self, rows: int, width: int, pages: int, block: int, cache: np.ndarray | None = None):
        self.table = np.full((rows, width), -1, np.int32)
        self.lens = np.zeros(rows, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.free = list(range(pages - 1, -1, -1))
        self.block, self.pages, self.width, self.rows = block, pages, width, rows
        self.cache = cache
        self.error = 0

    def _npages(self, tokens: int) -> int:
        return -(-int(tokens) // self.block)

    def resize(self, rows, lens, refused=()) -> list[int]:
        rows, lens = [int(r) for r in rows], [int(x) for x in lens]
        valid = [0 <= r < self.rows and rows.count(r) == 1 and x >= 0 and self._npages(x) <= self.width
                 for r, x in zip(rows, lens)]
        if not all(ok or i in refused for i, ok in enumerate(valid)):
            self.error |= ERR_ROW
        dropped = []
        for r, x, ok in zip(rows, lens, valid):
            if ok:
                dropped += self.table[r, self._npages(x):self._npages(self.lens[r])].tolist()
        last = {}
        for at, p in enumerate(dropped):
            if not 0 <= p < self.pages:
                self.error |= ERR_PAGE
            elif self.refs[p] > 0:
                self.refs[p] -= 1
                last[p] = at
            else:
                self.error |= ERR_REFS
        self.free += [p for p, _ in sorted(last.items(), key=lambda e: e[1]) if self.refs[p] == 0]
        have, asked, status = len(self.free), 0, []
        for r, x, ok in zip(rows, lens, valid):
            if not ok:
                status.append(INVALID)
                continue
            old, new = self._npages(self.lens[r]), self._npages(x)
            need = max(new - old, 0)
            asked += need
            if need and asked > have:
                status.append(NO_PAGES)
                continue
            for k in range(need):
                p = self.free.pop()
                self.table[r, old + k] = p
                if 0 <= p < self.pages:
                    self.refs[p] = 1
                else:                       # the free list was wrong: the row has it as it stands
                    self.error |= ERR_PAGE
            self.lens[r] = x
            status.append(OK)
        return status

    def copy(self, src, dst, tokens=None) -> None:
        for i, (a, b) in enumerate(zip(src, dst)):
            n = self.block if tokens is None else min(max(int(tokens[i]), 0), self.block)
            if n == 0 or a == b:
                continue
            if not (0 <= a < self.pages and 0 <= b < self.pages):
                self.error |= ERR_PAGE
                continue
            self.cache[:, b, :n] = self.cache[:, a, :n]

    def fork(self, parents, children) -> list[int]:
        parents, children = [int(p) for p in parents], [int(c) for c in children]
        have, asked, status = len(self.free), 0, []
        empty = self.lens == 0
        for p, c in zip(parents, children):
            if not (0 <= p < self.rows and 0 <= c < self.rows and children.count(c) == 1 and c not in parents and empty[c]):
                self.error |= ERR_ROW
                status.append(INVALID)
                continue
            if any(not 0 <= page < self.pages for page in self.table[p, :self._npages(self.lens[p])]):
                self.error |= ERR_PAGE
                status.append(INVALID)
                continue
            full, tail = divmod(int(self.lens[p]), self.block)
            asked += tail > 0
            if tail and asked > have:
                status.append(NO_PAGES)
                continue
            if tail and not 0 <= self.free[-1] < self.pages:
                self.free.pop()
                self.error |= ERR_PAGE
                status.append(INVALID)
                continue
            self.table[c, :full] = self.table[p, :full]
            for page in self.table[p, :full]:
                self.refs[page] += 1
            if tail:
                page = self.free.pop()
                self.table[c, full] = page
                self.refs[page] = 1
                self.copy([self.table[p, full]], [page], [tail])
            self.lens[c] = self.lens[p]
            status.append(OK)
        return status

    def _slot(self, r: int, pos: int):
        return int(self.table[r, pos // self.block]), pos % self.block

    def compact(self, rows, start, keep, offsets) -> list[int]:
        to, refused = [], set()
        rows = [int(r) for r in rows]
        for i, r in enumerate(rows):
            s, o0, o1 = int(start[i]), int(offsets[i]), int(offsets[i + 1])
            bad = 0
            if not 0 <= r < self.rows or rows.count(r) > 1:
                bad |= ERR_ROW
            length = int(self.lens[r]) if 0 <= r < self.rows else 0
            if not (0 <= o0 <= o1 <= len(keep)) or not 0 <= s <= length:
                bad |= ERR_KEEP
            if not bad:
                mine = [int(x) for x in keep[o0:o1]]
                if any(x <= (mine[j - 1] if j else s - 1) or x >= length for j, x in enumerate(mine)):
                    bad |= ERR_KEEP
            if not bad:
                moves = [(x, s + j) for j, x in enumerate(mine) if x != s + j]
                for _, t in moves:
                    if self.refs[self._slot(r, t)[0]] != 1:
                        bad |= ERR_REFS
            if bad:
                self.error |= bad
                refused.add(i)
                to.append(-1)
                continue
            for x, t in moves:
                a, b = self._slot(r, x), self._slot(r, t)
                self.cache[:, b[0], b[1]] = self.cache[:, a[0], a[1]]
            to.append(s + len(mine))
        return self.resize(rows, to, refused)
