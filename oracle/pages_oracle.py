"""The page books of a cache, kept one sequence and one page at a time: what the kernels that
fork, grow, free and compact on the GPU have to arrive at, number for number."""
import numpy as np


class Books:
    """refs [pages] and table [batch][max_pages] as Python lists."""

    def __init__(self, refs, table, block):
        self.refs = [int(n) for n in refs]
        self.table = [[int(p) for p in row] for row in table]
        self.block = block

    def _is_page(self, p):
        return 0 <= p < len(self.refs)

    def fork(self, lens, parents, children):
        for a, b in zip(parents, children):
            if a == b or not (0 <= a < len(self.table) and 0 <= b < len(self.table)):
                continue
            n = -(-max(int(lens[a]), 0) // self.block)
            row = [p if e < n and self._is_page(p) else -1 for e, p in enumerate(self.table[a])]
            self.table[b] = row
            for p in row:
                if p >= 0:
                    self.refs[p] += 1

    def free(self, rows=None):
        for b in range(len(self.table)) if rows is None else rows:
            if not 0 <= b < len(self.table):
                continue
            for p in self.table[b]:
                if self._is_page(p):
                    self.refs[p] -= 1
            self.table[b] = [-1] * len(self.table[b])

    def grow(self, filled, new):
        """(src, dst, missing); who holds a page is read before anything is handed out."""
        before = list(self.refs)
        free = [p for p, n in enumerate(before) if n <= 0]
        out = bool(False)  # a sequence has wanted more than there were
        src, dst, missing = [], [], []
        for b, row in enumerate(self.table):
            src.append(-1)
            dst.append(-1)
            missing.append(0)
            held, n = max(int(filled[b]), 0), int(new[b])
            if n <= 0:
                continue
            first, last = held // self.block, (held + n - 1) // self.block
            part = held % self.block > 0
            wants = []
            for e in range(first, min(last + 1, len(row))):
                if self._is_page(row[e]):
                    if before[row[e]] > 1:
                        wants.append(e)
                elif not (part and e == first):
                    wants.append(e)
            past = max(0, last + 1 - max(first, len(row)))
            if past:
                missing[b] = len(wants) + past
                continue
            if wants and (out or len(wants) > len(free)):
                out = True
                missing[b] = len(wants)
                continue
            for e in wants:
                page, old = free.pop(0), row[e]
                row[e] = page
                self.refs[page] = 1
                if self._is_page(old):
                    self.refs[old] -= 1
                    if part and e == first:
                        src[b], dst[b] = old, page
        return src, dst, missing

    def compact(self):
        """(src, dst, used), padded as the operator pads."""
        pages = len(self.refs)
        used = sum(n > 0 for n in self.refs)
        holes = [p for p in range(used) if self.refs[p] <= 0]
        moved = [p for p in range(used, pages) if self.refs[p] > 0]
        to = dict(zip(moved, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        pad = [-1] * (pages // 2 - len(moved))
        return moved + pad, holes + pad, used

    def same(self, refs, table):
        return (np.array_equal(np.asarray(self.refs), refs)
                and np.array_equal(np.asarray(self.table).reshape(table.shape), table))
