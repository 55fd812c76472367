"""A paged cache restated in plain Python: what the page_* calls do to the tables and the pages, one
list entry after the other."""
from __future__ import annotations

import torch


class Model:
    def __init__(self, buffers, n_pages, page, max_seqs, width):
        self.buffers = [b.clone().cpu() for b in buffers]
        self.n_pages, self.page, self.width = n_pages, page, width
        self.table = [[-1] * width for _ in range(max_seqs)]
        self.lens = [0] * max_seqs
        self.refs = [0] * n_pages
        self.status = [0, 0]

    def _pages(self, n):
        return -(-n // self.page)

    def extend(self, seqs, counts):
        """Slots of the new tokens, entry by entry."""
        free = [p for p, r in enumerate(self.refs) if r == 0]
        slots, seen, cum = [], set(), 0
        for s, c in zip(seqs, counts):
            first = s not in seen
            seen.add(s)
            if s < 0:
                slots += [-1] * c
                continue
            if not first or s >= len(self.lens) or self._pages(self.lens[s] + c) > self.width:
                self.status[0] += 1
                slots += [-1] * c
                continue
            old, have = self.lens[s], self._pages(self.lens[s])
            need = self._pages(old + c) - have
            cum += need
            if need and cum > len(free):
                self.status[0] += 1
                self.status[1] += need
                slots += [-1] * c
                continue
            for k in range(need):
                p = free[cum - need + k]
                self.table[s][have + k] = p
                self.refs[p] = 1
            self.lens[s] = old + c
            slots += [self.table[s][i // self.page] * self.page + i % self.page for i in range(old, old + c)]
        return slots

    def write(self, rows, slots):
        for b, r in zip(self.buffers, rows):
            r = r.cpu()
            for t, slot in enumerate(slots):
                if 0 <= slot < self.n_pages * self.page:
                    b[slot // self.page, slot % self.page] = r[t]

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.lens):
                for m, p in enumerate(self.table[s]):
                    if p >= 0:
                        self.refs[p] -= 1
                        self.table[s][m] = -1
                self.lens[s] = 0

    def fork(self, src, dst):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        table, lens, before = [row[:] for row in self.table], self.lens[:], [b.clone() for b in self.buffers]
        named, done, taken = set(), [], 0
        for s, d in zip(src, dst):
            if s < 0 or d < 0:
                continue
            if s >= len(lens) or d >= len(lens) or d in named:
                self.status[0] += 1
                continue
            named.add(d)
            if s == d:
                continue
            full, tail = divmod(lens[s], self.page)
            row = table[s][:full] + [-1] * (self.width - full)
            if tail:
                taken += 1
                if taken > len(free):
                    self.status[0] += 1
                    self.status[1] += 1
                    continue
                row[full] = free[taken - 1]
                self.refs[row[full]] = 1
                for b, old in zip(self.buffers, before):
                    b[row[full], :tail] = old[table[s][full], :tail]
            for p in row[:full]:
                self.refs[p] += 1
            done.append((d, row, lens[s]))
        for d, row, n in done:
            for p in table[d]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[d], self.lens[d] = row, n

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        out = [p for p in range(live, self.n_pages) if self.refs[p] > 0]
        holes = [p for p in range(live) if self.refs[p] == 0]
        to = dict(zip(out, holes))
        for p, q in to.items():
            self.refs[q], self.refs[p] = self.refs[p], 0
            for b in self.buffers:
                b[q] = b[p]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return live, len(out)

    def rows_of(self, s, buffer):
        """The rows of sequence s in position order."""
        at = [self.table[s][i // self.page] for i in range(self.lens[s])]
        return torch.stack([self.buffers[buffer][p, i % self.page] for i, p in enumerate(at)]) if at else None

    def assert_same(self, table, lens, refs, status, buffers):
        assert lens.tolist() == self.lens
        assert table.tolist() == self.table
        assert refs.tolist() == self.refs
        assert status.tolist() == self.status
        for k, (got, want) in enumerate(zip(buffers, self.buffers)):
            got, want = got.cpu(), want
            raw = lambda t: t.contiguous().view(torch.uint8)
            assert torch.equal(raw(got), raw(want)), f"buffer {k} differs"

    def assert_consistent(self):
        count = [0] * self.n_pages
        for row in self.table:
            for p in row:
                if p >= 0:
                    count[p] += 1
        assert count == self.refs
