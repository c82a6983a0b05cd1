"""A cache in pages, plainly: lists and numpy in 64 bits, one position at a time. What ytensor_b200.paged is held to."""
import math

import numpy as np

FULL, INVALID, SHARED = 1, 2, 4


class PlainPages:
    """k, v [layers, pages, heads, page, dim] in float64; table, held, lens and refs as lists."""

    def __init__(self, layers, pages, page, heads, dim, slots, max_pages):
        self.k = np.full((layers, pages, heads, page, dim), np.nan)
        self.v = self.k.copy()
        self.layers, self.pages, self.page, self.heads, self.dim = layers, pages, page, heads, dim
        self.table, self.max_pages = [[] for _ in range(slots)], max_pages
        self.lens, self.refs, self.status = [0] * slots, [0] * pages, 0

    @property
    def slots(self):
        return len(self.lens)

    @property
    def held(self):
        return [len(t) for t in self.table]

    def _pages(self, n):
        return -(-n // self.page)

    def row(self, slot, at):
        """(page, row) of a position; None where the slot holds no page."""
        i = at // self.page
        return (self.table[slot][i], at % self.page) if 0 <= i < len(self.table[slot]) else None

    def reserve(self, counts):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        want = []
        for s, n in enumerate(counts):
            if n <= 0:
                if n < 0:
                    self.status |= INVALID
                continue
            if self._pages(self.lens[s] + n) > self.max_pages:
                self.status |= FULL
                return
            at = self.lens[s] // self.page
            if self.lens[s] % self.page and self.refs[self.table[s][at]] > 1:
                want.append((s, at))
            want += [(s, i) for i in range(len(self.table[s]), self._pages(self.lens[s] + n))]
        if len(want) > len(free):
            self.status |= FULL
            return
        for (s, i), new in zip(want, free):
            if i < len(self.table[s]):
                old, rows = self.table[s][i], self.lens[s] % self.page
                for pool in (self.k, self.v):
                    pool[:, new, :, :rows] = pool[:, old, :, :rows]
                self.refs[old] -= 1
                self.table[s][i] = new
            else:
                self.table[s].append(new)
            self.refs[new] = 1

    def fork(self, source):
        old, lens = [list(t) for t in self.table], list(self.lens)
        for s, a in enumerate(source):
            if a == s:
                continue
            if not -1 <= a < self.slots:
                self.status |= INVALID
                continue
            self.table[s] = [] if a < 0 else old[a][:self._pages(lens[a])]
            self.lens[s] = 0 if a < 0 else lens[a]
        self.refs = [0] * self.pages
        for t in self.table:
            for p in t:
                self.refs[p] += 1

    def append(self, layer, k, v, starts):
        for s in range(self.slots):
            for i in range(starts[s + 1] - starts[s]):
                at = self.row(s, self.lens[s] + i)
                if at is None:
                    self.status |= INVALID
                elif self.refs[at[0]] != 1:
                    self.status |= SHARED
                else:
                    self.k[layer, at[0], :, at[1]] = k[starts[s] + i]
                    self.v[layer, at[0], :, at[1]] = v[starts[s] + i]

    def keep(self, kept, accepted=None, base=None):
        base = list(self.lens if base is None else base)
        for s in range(self.slots):
            row = list(range(kept[s])) if accepted is None else list(accepted[s][:kept[s]])
            places = [base[s] + j for j in range(len(row))] + [base[s] + a for a in row]
            if (kept[s] < 0 or len(row) < kept[s] or any(a <= b for a, b in zip(row, [-1] + row)) or
                    any(self.row(s, p) is None for p in places) or base[s] + kept[s] > len(self.table[s]) * self.page):
                self.status |= INVALID
                continue
            if any(a != j and self.refs[self.row(s, base[s] + j)[0]] != 1 for j, a in enumerate(row)):
                self.status |= SHARED
                continue
            for j, a in enumerate(row):
                x, y = self.row(s, base[s] + a), self.row(s, base[s] + j)
                for pool in (self.k, self.v):
                    pool[:, y[0], :, y[1]] = pool[:, x[0], :, x[1]].copy()
            self.lens[s] = base[s] + kept[s]

    def compact(self, into):
        live = [p for p, r in enumerate(self.refs) if r]
        if len(live) > into.pages:
            into.status |= FULL
            return
        number = {p: i for i, p in enumerate(live)}
        into.table = [[number[p] for p in t] for t in self.table]
        into.lens = list(self.lens)
        into.refs = [self.refs[p] for p in live] + [0] * (into.pages - len(live))
        for name in ("k", "v"):
            getattr(into, name)[:, :len(live)] = getattr(self, name)[:, live]

    def attend(self, layer, q, starts, parents=None, k=None, v=None, scale=0.0):
        """(o, weighted mean of |v|, largest sum of |q||k| of a row's scores): the last two are what errors go by."""
        groups, scale = q.shape[1] // self.heads, scale or 1 / math.sqrt(self.dim)
        out, size, big = np.zeros(q.shape), np.zeros(q.shape), 1.0
        for s in range(self.slots):
            a, n, L = starts[s], starts[s + 1] - starts[s], self.lens[s]
            if not n:
                continue
            seen = np.zeros((n, L + n), bool)
            seen[:, :L] = True
            for i in range(n):
                j = i
                while j >= 0:
                    seen[i, L + j] = True
                    j = parents[a + j] if parents is not None else j - 1
            at = [self.row(s, p) for p in range(L if k is not None else L + n)]
            pg, row = np.array([x[0] for x in at], int), np.array([x[1] for x in at], int)
            for h in range(self.heads):
                K, V = self.k[layer, pg, h, row], self.v[layer, pg, h, row]
                if k is not None:
                    K, V = np.concatenate([K, k[a:a + n, h]]), np.concatenate([V, v[a:a + n, h]])
                for g in range(h * groups, (h + 1) * groups):
                    # (what a row does not see has no part in it, whatever stands there)
                    x = np.where(seen, q[a:a + n, g] @ np.nan_to_num(K).T * scale, -np.inf)
                    p = np.exp(x - x.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    out[a:a + n, g], size[a:a + n, g] = p @ np.nan_to_num(V), p @ np.abs(np.nan_to_num(V))
                    big = max(big, float((np.abs(q[a:a + n, g]) @ np.abs(np.nan_to_num(K)).T).max() * abs(scale)))
        return out, size, big
