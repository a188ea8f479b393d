"""Plain restatements of the search and history operators, for the tests: numpy in
64 bits for the selections, Python lists for the paged history."""

from __future__ import annotations

import numpy as np

HEADS = (3, 3, 3, 2, 2, 3, 2)


def best_continuations(logits, scores, mask, finished, width, heads=None):
    """scores (float64), parents, actions of the `width` best per group; logits [G, K, V]."""
    G, K, V = logits.shape
    heads = heads or (V,)
    size = int(np.prod(heads))
    x, s = logits.astype(np.float64), scores.astype(np.float64)
    out_s = np.full((G, width), -np.inf)
    out_p = np.tile(np.arange(width) % K, (G, 1))
    out_a = np.zeros((G, width), np.int64)
    for g in range(G):
        totals = np.full((K, size), -np.inf)
        for k in range(K):
            if not s[g, k] > -np.inf:
                continue
            if finished is not None and finished[g, k]:
                totals[k, 0] = s[g, k]
                continue
            sums, norm, at, bad = np.zeros(1), 0.0, 0, False
            for h in heads:
                row = x[g, k, at:at + h]
                ok = np.ones(h, bool) if mask is None else mask[g, k, at:at + h]
                row = np.where(ok, row, -np.inf)
                bad |= bool(np.isnan(row).any() or (row == np.inf).any() or not (row > -np.inf).any())
                if not bad:
                    norm += row.max() + np.log(np.exp(row - row.max()).sum())
                sums = np.add.outer(sums, row).ravel()
                at += h
            if not bad:
                totals[k] = (s[g, k] - norm) + sums
        flat = totals.ravel()
        live = np.nonzero(flat > -np.inf)[0]
        if live.size > width:
            live = live[flat[live] >= np.partition(flat[live], live.size - width)[live.size - width]]
        order = live[np.lexsort((live, -flat[live]))][:width]
        out_s[g, :order.size] = flat[order]
        out_p[g, :order.size] = order // size
        out_a[g, :order.size] = order % size
    return out_s, out_p, out_a


def joint_actions(index):
    return np.stack(np.unravel_index(index, HEADS), -1)


class ListHistory:
    """The paged history with one Python step per row."""

    def __init__(self, pages, table, lengths, refs):
        self.pages, self.table = pages.copy(), table.copy()
        self.lengths, self.refs, self.dropped = lengths.copy(), refs.copy(), 0

    def page(self, r, c):
        p = int(self.table[r, c])
        return p if 0 <= p < len(self.refs) else -1

    def fork(self, parents):
        P, M = self.pages.shape[1], self.table.shape[1]
        new = ListHistory(self.pages, np.full((len(parents), M), -1, np.int32), np.zeros(len(parents), np.int32),
                          np.zeros_like(self.refs))
        new.dropped = self.dropped
        for r, q in enumerate(parents):
            if not 0 <= q < len(self.lengths):
                continue
            new.lengths[r] = self.lengths[q]
            for c in range(min(M, -(-max(0, int(self.lengths[q])) // P))):
                new.table[r, c] = self.page(q, c)
                if new.table[r, c] >= 0:
                    new.refs[new.table[r, c]] += 1
        return new

    def append(self, records, mask=None):
        P, M = self.pages.shape[1], self.table.shape[1]
        rows = [r for r in range(len(self.lengths)) if mask is None or mask[r]]
        share = {}
        for r in rows:
            c, slot = divmod(int(self.lengths[r]), P)
            if c < M and slot > 0 and self.page(r, c) >= 0 and self.refs[self.page(r, c)] > 1:
                share.setdefault(self.page(r, c), []).append((-slot, r))
        stays = {min(rs)[1] for p, rs in share.items() if len(rs) == self.refs[p]}
        copies = {r for rs in share.values() for _, r in rs} - stays
        free = iter([p for p in range(len(self.refs)) if self.refs[p] <= 0])
        before = self.pages.copy()
        for r in rows:
            c, slot = divmod(int(self.lengths[r]), P)
            if c >= M or (slot > 0 and self.page(r, c) < 0):
                self.dropped += 1
                continue
            if slot == 0 or r in copies:
                p = next(free, None)
                if p is None:
                    self.dropped += 1
                    continue
                if r in copies:
                    old = self.page(r, c)
                    self.pages[p, :slot] = before[old, :slot]
                    self.refs[old] -= 1
                self.refs[p] = 1
                self.table[r, c] = p
            self.pages[self.table[r, c], slot] = records[r]
            self.lengths[r] += 1

    def free(self, mask):
        for r in np.nonzero(mask)[0]:
            for c in range(self.table.shape[1]):
                if self.page(r, c) >= 0:
                    self.refs[self.page(r, c)] -= 1
            self.table[r] = -1
            self.lengths[r] = 0

    def compact(self):
        live = [p for p in range(len(self.refs)) if self.refs[p] > 0]
        holes = [p for p in range(len(live)) if self.refs[p] <= 0]
        for to, old in zip(holes, reversed([p for p in live if p >= len(live)])):
            self.pages[to] = self.pages[old]
            self.refs[to], self.refs[old] = self.refs[old], 0
            self.table[self.table == old] = to
        return len(live)

    def read(self, steps, rows):
        P, M = self.pages.shape[1], self.table.shape[1]
        out = np.zeros((len(rows), steps) + self.pages.shape[2:], self.pages.dtype)
        counts = np.zeros(len(rows), np.int32)
        for i, r in enumerate(rows):
            n = min(max(0, int(self.lengths[r])), M * P) if 0 <= r < len(self.lengths) else 0
            counts[i] = min(n, steps)
            for t in range(counts[i]):
                at = n - counts[i] + t
                p = self.page(r, at // P)
                if p >= 0:
                    out[i, t] = self.pages[p, at % P]
        return out, counts
