"""Plain models of the batch tables: a page pool whose streams append different numbers
of frames, stream after stream, and the grouping of rows by adapter."""

from collections import deque

import numpy as np


class RaggedPool:
    """Pages of every slot by logical number, the free ones in a FIFO queue."""

    def __init__(self, num_slots, page_size, left, chunk, order):
        self.P, self.window, self.chunk = page_size, left + chunk, chunk
        self.M = (self.window + page_size - 2) // page_size + 1
        self.free = deque(int(p) for p in order)
        self.A = [0] * num_slots
        self.held = [dict() for _ in range(num_slots)]

    def ring(self, s):
        r = np.full(self.M, -1, dtype=np.int32)
        for k, page in self.held[s].items():
            assert r[k % self.M] == -1
            r[k % self.M] = page
        return r

    def advance(self, slots, lengths):
        rows = np.full((len(slots), 1 + self.M), -1, dtype=np.int32)
        rows[:, 0] = 0
        place = np.full((len(slots), self.chunk), -1, dtype=np.int32)
        seen = set()
        for b, (s, n) in enumerate(zip(slots, lengths)):
            if not 0 <= s < len(self.A) or s in seen:
                continue
            seen.add(s)
            n = min(max(int(n), 0), self.chunk)
            a, held = self.A[s], self.held[s]
            for k in sorted(held):
                if (k + 1) * self.P <= a + n - self.window:
                    self.free.append(held.pop(k))
            for t in range(n):
                k = (a + t) // self.P
                if k not in held:
                    held[k] = self.free.popleft()
                place[b, t] = held[k] * self.P + (a + t) % self.P
            rows[b, 0], rows[b, 1:] = a, self.ring(s)
            self.A[s] = a + n
        return rows, place

    def reset(self, slots):
        seen = set()
        for s in slots:
            if 0 <= s < len(self.A) and s not in seen:
                seen.add(s)
                self.free.extend(self.held[s][k] for k in sorted(self.held[s]))
                self.held[s], self.A[s] = {}, 0


def plan_model(ids, frames, bank):
    """(order, sorted ids, tiles) of the rows by adapter."""
    key = np.where((ids >= 0) & (ids < bank), ids, bank).repeat(frames)
    order = np.argsort(key, kind="stable")
    key = key[order]
    tiles, n = [], len(key) // 32 + min(bank, len(ids))
    for g in range(bank):
        at = np.flatnonzero(key == g)
        tiles += [[g, at[i], min(32, len(at) - i), 0] for i in range(0, len(at), 32)]
    assert len(tiles) <= n
    tiles += [[-1, 0, 0, 0]] * (n - len(tiles))
    return order, np.where(key < bank, key, -1), np.array(tiles).reshape(-1, 4)
