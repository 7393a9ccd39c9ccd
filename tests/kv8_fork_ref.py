"""A plain pool of pages that several sequences may hold, by the order that the header states."""
import numpy as np

import kv8_ref
from kv8_ref import BLOCK


class SharedPool(kv8_ref.Pool):
    def __init__(self, seqs, max_len, pages):
        super().__init__(seqs, max_len, pages)
        self.pages, self.lens = pages, [0] * seqs

    def holders(self):
        n = [0] * self.pages
        for t in self.tables:
            for p in t:
                n[p] += 1
        return n

    def plan(self, have, add, rows):
        """As Pool.plan; None, too, where rows would lie in a page that others hold afterwards."""
        need = [-(-(h + a) // BLOCK) for h, a in zip(have, add)]
        if min(have) < 0 or min(add) < 0 or max(h + a for h, a in zip(have, add)) > self.max_len or sum(add) > rows:
            return None
        after = self.holders()
        gone = [p for t, n in zip(self.tables, need) for p in t[n:]]
        for p in gone:
            after[p] -= 1
        for t, h, a, n in zip(self.tables, have, add, need):
            if a and any(after[p] > 1 for p in t[h // BLOCK:n]):
                return None
        back = [p for i, p in enumerate(gone) if after[p] == 0 and p not in gone[:i]]
        if sum(max(n - len(t), 0) for t, n in zip(self.tables, need)) > len(self.stack) + len(back):
            return None
        self.lens = [h + a for h, a in zip(have, add)]
        for t, n in zip(self.tables, need):
            del t[n:]
        self.stack += back
        return super().plan(have, add, rows) if sum(need) <= sum(map(len, self.tables)) + len(self.stack) else self._take(have, add, need)

    def _take(self, have, add, need):
        for t, n in zip(self.tables, need):
            while len(t) < n:
                t.append(self.stack.pop())
        starts = np.concatenate([[0], np.cumsum(add)])
        seq = [b for b, a in enumerate(add) for _ in range(a)]
        pos = [h + i for h, a in zip(have, add) for i in range(a)]
        slots = [self.tables[b][p // BLOCK] * BLOCK + p % BLOCK for b, p in zip(seq, pos)]
        return starts, np.array(pos, int), np.array(slots, int), self.table(), np.array(seq, int)

    def table(self):
        t = np.full((len(self.tables), self.W), -1)
        for b, pages in enumerate(self.tables):
            t[b, :len(pages)] = pages
        return t

    def fork(self, source, keep):
        """The copied pages [(from, to)], or None, when nothing changes."""
        B = len(self.tables)
        for f, k in zip(source, keep):
            if k < 0 or (k and (not 0 <= f < B or k > self.lens[f])):
                return None
        tables = [list(self.tables[f][:-(-k // BLOCK)]) if k else [] for f, k in zip(source, keep)]
        whole = {p for t, k in zip(tables, keep) for p in t[:k // BLOCK]}
        held = {p for t in tables for p in t}
        free = [p for p in range(self.pages) if p not in held]
        kept, copies = set(), []
        for b, k in enumerate(keep):
            if k % BLOCK == 0:
                continue
            p = tables[b][-1]
            if p in whole or p in kept:
                copies.append((b, p))
            else:
                kept.add(p)
        if len(copies) > len(free):
            return None
        for (b, _), to in zip(copies, free):
            tables[b][-1] = to
        self.tables, self.lens = tables, list(keep)
        self.stack = free[len(copies):][::-1]
        return [(p, to) for (_, p), to in zip(copies, free)]
