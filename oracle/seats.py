"""The seats' books seat by seat and page by page, from their definition (test infrastructure; csrc/seats_step.hip is checked against it)."""

from __future__ import annotations


class Books:
    def __init__(self, lens, table, free, left, keys, page, rows, text):
        """text: positions that each content takes"""
        self.lens, self.table, self.stack = list(map(int, lens)), [list(map(int, t)) for t in table], list(map(int, free[:left]))
        self.keys, self.page, self.rows, self.text = keys, page, rows, list(map(int, text))

    def step(self, new, drop, content):
        """-> slots, positions, first, took"""
        page, back = self.page, []
        for r, n in enumerate(self.lens):
            stay = n - min(max(int(drop[r]), 0), n)
            back += self.table[r][-(-stay // page) : -(-n // page)]
            self.lens[r] = stay
        self.stack += reversed(back)
        have, tokens, pages = len(self.stack), 0, 0
        slots, pos, first, took = [], [], [0], []
        for r, m in enumerate(map(int, new)):
            n = self.lens[r]
            m = m if 0 < m <= self.keys - n else 0
            need = -(-(n + m) // page) - -(-n // page)
            tokens, pages = tokens + m, pages + need
            if tokens > self.rows or (need and pages > have):
                m = need = 0
            for i in range(need):
                self.table[r][-(-n // page) + i] = self.stack.pop()
            c = int(content[r])
            for s in range(n, n + m):
                slots.append(self.table[r][s // page] * page + s % page)
                pos.append(s + (self.text[c] if 0 <= c < len(self.text) else 0))
            self.lens[r] = n + m
            took.append(m)
            first.append(len(slots))
        pad = self.rows - len(slots)
        return slots + [-1] * pad, pos + [0] * pad, first, took
