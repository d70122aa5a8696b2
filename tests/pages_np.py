"""The page operations on host arrays, entry by entry."""
import numpy as np


class Pages:
    """Tables of a pool: page_table, kv_len, refs, and the layers' pools [(keys, values), ...] [pages][kv_heads][page][...]."""

    def __init__(self, table, kv_len, refs, page, layers=(), prefix=0, prefix_pages=()):
        self.table, self.kv_len, self.refs = np.array(table, np.int32), np.array(kv_len, np.int64), np.array(refs, np.int32)
        self.page, self.layers, self.prefix, self.prefix_pages = page, [tuple(x.copy() for x in l) for l in layers], prefix, np.array(prefix_pages, np.int32)

    def held(self, e):
        return 0 <= e < len(self.refs)

    def take(self, free):
        """The lowest free page of those that the call found."""
        return free.pop(0) if free else -1

    def free(self):
        return [p for p in range(len(self.refs)) if self.refs[p] <= 0]

    def reserve(self, want):
        lacking, free = 0, self.free()
        for s, n in enumerate(want):
            entries = -(-max(0, int(n) - self.prefix) // self.page)
            lacking += entries > self.table.shape[1]
            for e in range(min(entries, self.table.shape[1])):
                if not self.held(self.table[s, e]):
                    p = self.take(free)
                    if p < 0:
                        lacking += 1
                    else:
                        self.table[s, e], self.refs[p] = p, 1
        return lacking

    def fork(self, parents, children):
        lacking, free = 0, self.free()
        before = self.table.copy()
        for p, c in zip(parents, children):
            if not (0 <= p < len(self.kv_len) and 0 <= c < len(self.kv_len)) or p == c:
                continue
            full, slots = divmod(max(0, int(self.kv_len[p]) - self.prefix), self.page)
            full, slots = (full, slots) if full < self.table.shape[1] else (self.table.shape[1], 0)
            last = before[p, full] if slots else -1
            self.table[c] = -1
            if self.held(last):
                got = self.take(free)
                if got < 0:
                    lacking += 1
                    self.kv_len[c] = 0
                    continue
                self.table[c, full], self.refs[got] = got, 1
                for k, v in self.layers:
                    for x in (k, v):
                        self.copy_slots(x, got, last, slots)
            for e in range(full):
                if self.held(before[p, e]):
                    self.table[c, e] = before[p, e]
                    self.refs[before[p, e]] += 1
            self.kv_len[c] = self.kv_len[p]
        return lacking

    def copy_slots(self, x, dst, src, slots):
        if x.dtype == np.uint8:              # codes of all slots, then their scales
            hd = x.shape[-1] // 17 * 32
            for h in range(x.shape[1]):
                d, s = x[dst, h].reshape(-1), x[src, h].reshape(-1)
                d[:slots * hd // 2] = s[:slots * hd // 2]
                at = self.page * hd // 2
                d[at:at + slots * hd // 32] = s[at:at + slots * hd // 32]
        else:
            x[dst, :, :slots] = x[src, :, :slots]

    def release(self, seqs):
        for s in seqs:
            if not 0 <= s < len(self.kv_len):
                continue
            for e in self.table[s]:
                if self.held(e):
                    self.refs[e] -= 1
            self.table[s] = -1
            self.kv_len[s] = 0

    def compact(self):
        used = int((self.refs > 0).sum())
        holes = [p for p in range(used) if self.refs[p] <= 0]
        moves = dict(zip([p for p in range(used, len(self.refs)) if self.refs[p] > 0], holes))
        for src, dst in moves.items():
            for k, v in self.layers:
                for x in (k, v):
                    x[dst] = x[src]
            self.refs[dst], self.refs[src] = self.refs[src], 0
        for t in (self.table, self.prefix_pages):
            for i, e in np.ndenumerate(t):
                t[i] = moves.get(int(e), e)
        return used

    def check(self):
        """Every page's references are the entries that name it."""
        count = np.zeros(len(self.refs), int)
        for e in (*self.table.ravel(), *self.prefix_pages):
            if self.held(e):
                count[e] += 1
        assert np.array_equal(np.maximum(self.refs, 0), count)
