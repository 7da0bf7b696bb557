"""A paged cache in plain Python, call by call as include/whisper4j_cuda.h defines them."""
import numpy as np


class PagesRef:
    def __init__(self, pool, ref, table, length):
        self.pool, self.ref, self.table, self.len = (np.array(a) for a in (pool, ref, table, length))
        self.page = self.pool.shape[3]

    def held(self, row):
        return [int(p) for p in self.table[row, :-(-int(self.len[row]) // self.page)]]

    def _free(self):
        return [i for i, n in enumerate(self.ref) if n == 0]

    def fork(self, dst, src):
        old = {r: (self.held(r), int(self.len[r])) for r in set(dst) | set(src) if r >= 0}
        free, goes_on = self._free(), {r: r not in dst or src[dst.index(r)] == r for r in old}
        taken = set()
        for d, s in zip(dst, src):
            if d == s:
                continue
            for p in old[d][0]:
                self.ref[p] -= 1
        for d, s in zip(dst, src):
            if d == s:
                continue
            pages, n = old[s] if s >= 0 else ([], 0)
            pages = list(pages)
            if n % self.page:
                if goes_on[s] or s in taken:
                    mine = free.pop(0)
                    self.pool[:, mine, :, :n % self.page] = self.pool[:, pages[-1], :, :n % self.page]
                    pages[-1] = mine
                taken.add(s)
            for j, p in enumerate(pages):
                self.table[d, j] = p
                self.ref[p] += 1
            self.len[d] = n

    def free(self, rows):
        for r in rows:
            for p in self.held(r):
                self.ref[p] -= 1
            self.len[r] = 0

    def extend(self, rows, start):
        free = self._free()
        for i, r in enumerate(rows):
            had = len(self.held(r))
            self.len[r] += start[i + 1] - start[i]
            for j in range(had, -(-int(self.len[r]) // self.page)):
                self.table[r, j] = free.pop(0)
                self.ref[self.table[r, j]] = 1

    def write(self, layer, rows, start, k, v):
        for i, r in enumerate(rows):
            for t in range(start[i], start[i + 1]):
                at = int(self.len[r]) - start[i + 1] + t
                page = self.table[r, at // self.page]
                self.pool[2 * layer, page, :, at % self.page] = k[t]
                self.pool[2 * layer + 1, page, :, at % self.page] = v[t]

    def compact(self):
        live = int((self.ref > 0).sum())
        holes = [i for i in range(live) if self.ref[i] == 0]
        high = [i for i in range(live, len(self.ref)) if self.ref[i] > 0]
        to = dict(zip(high, holes))
        for h, p in to.items():
            self.pool[:, p] = self.pool[:, h]
            self.ref[p], self.ref[h] = self.ref[h], 0
        for r in range(len(self.len)):
            for j, p in enumerate(self.held(r)):
                self.table[r, j] = to.get(p, p)
        return live
