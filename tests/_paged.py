"""A paged cache in plain numpy: the page operations done one after another on
the host, attention in 64 bits, and the bound its 16-bit kernels keep."""
from __future__ import annotations

import numpy as np


class Pages:
    """Page table, lengths, reference counts and contents [planes][pages][elems]."""

    OK, SHORT, BAD = 0, 1, 2

    def __init__(self, pool, rows, stride, page_size):
        self.pool = pool
        self.table = np.full((rows, stride), -1, np.int32)
        self.len = np.zeros(rows, np.int32)
        self.ref = np.zeros(pool.shape[1], np.int32)
        self.ps = page_size

    def held(self, n):
        return -(-int(n) // self.ps)

    def _items(self, seqs):
        live = [s for s in seqs if s >= 0]
        return len(set(live)) == len(live) and all(s < len(self.len) for s in live)

    def truncate(self, seqs, new_len=None):
        new_len = [0] * len(seqs) if new_len is None else new_len
        if not self._items(seqs) or any(s >= 0 and not 0 <= n <= self.len[s] for s, n in zip(seqs, new_len)):
            return self.BAD
        for s, n in zip(seqs, new_len):
            if s < 0:
                continue
            for j in range(self.held(n), self.held(self.len[s])):
                self.ref[self.table[s, j]] -= 1
                self.table[s, j] = -1
            self.len[s] = n
        return self.OK

    def fork(self, parents, children, fork_len=None):
        items = [(p, c, (int(self.len[p]) if p < len(self.len) else 0) if fork_len is None else fork_len[i])
                 for i, (p, c) in enumerate(zip(parents, children)) if p >= 0 and c >= 0]
        if not self._items([c for _, c, _ in items]):
            return self.BAD
        for p, c, n in items:
            if p >= len(self.len) or p == c or self.len[c] != 0 or not 0 <= n <= self.len[p]:
                return self.BAD
        for p, c, n in items:
            k = self.held(n)
            self.table[c, :k] = self.table[p, :k]
            for g in self.table[p, :k]:
                self.ref[g] += 1
        for _, c, n in items:
            self.len[c] = n
        return self.OK

    def extend(self, seqs, take):
        """(status, pages taken or None, first positions)"""
        none = np.full(len(seqs), -1, np.int32)
        cap = self.table.shape[1] * self.ps
        if not self._items(seqs) or any(s >= 0 and (t < 0 or self.len[s] + t > cap) for s, t in zip(seqs, take)):
            return self.BAD, None, none
        last = [int(self.table[s, self.held(self.len[s]) - 1]) if s >= 0 and t > 0 and self.len[s] % self.ps else -1
                for s, t in zip(seqs, take)]
        plan, need = [], 0
        for i, (s, t) in enumerate(zip(seqs, take)):
            if s < 0:
                plan.append(None)
                continue
            g = last[i]
            cow = g >= 0 and self.ref[g] > 1
            if cow and last.count(g) == self.ref[g] and last.index(g) == i:
                cow = False
            grow = self.held(self.len[s] + t) - self.held(self.len[s])
            plan.append((cow, grow))
            need += cow + grow
        free = [int(g) for g in np.nonzero(self.ref == 0)[0]]
        if need > len(free):
            return self.SHORT, need, none
        first = none.copy()
        for i, (s, t) in enumerate(zip(seqs, take)):
            if plan[i] is None:
                continue
            cow, grow = plan[i]
            k = self.held(self.len[s])
            if cow:
                g = free.pop(0)
                self.pool[:, g] = self.pool[:, last[i]]
                self.ref[last[i]] -= 1
                self.ref[g] = 1
                self.table[s, k - 1] = g
            for j in range(grow):
                g = free.pop(0)
                self.ref[g] = 1
                self.table[s, k + j] = g
            first[i] = self.len[s]
            self.len[s] += t
        return self.OK, need, first

    def compact(self):
        n = int((self.ref > 0).sum())
        src = [g for g in range(n, len(self.ref)) if self.ref[g] > 0]
        dst = [g for g in range(n) if self.ref[g] == 0]
        to = {}
        for s, d in zip(src, dst):
            self.pool[:, d] = self.pool[:, s]
            self.ref[d], self.ref[s] = self.ref[s], 0
            to[s] = d
        for s in range(len(self.len)):
            for j in range(self.held(self.len[s])):
                self.table[s, j] = to.get(int(self.table[s, j]), self.table[s, j])
        return n

    def check(self):
        """What holds after every operation."""
        count = np.zeros_like(self.ref)
        for s in range(len(self.len)):
            k = self.held(self.len[s])
            pages = self.table[s, :k]
            assert np.all(pages >= 0) and len(set(pages.tolist())) == k
            np.add.at(count, pages, 1)
        np.testing.assert_array_equal(count, self.ref)


def rows_of(pages, table_row, n, page_size):
    """Token rows 0..n-1 of a sequence from pages [num_pages][page_size][row]."""
    j = np.arange(n)
    return pages[table_row[j // page_size], j % page_size]


def attend64(q, k, v, heads, kv_heads):
    """softmax(q k / sqrt(d)) v in 64 bits; q [heads][d], k, v [n][kv_heads][d].
    Returns the output and a bound on the kernels' error at each element.

    The kernels multiply 16-bit operands and add in 32 bits, round a weight p
    to 16 bits (half a step, 2^-11 of it; 2^-25 where p is subnormal, p being
    at most 2^8 and their sum at least 1) and the output once (2^-11, 2^-25).
    A score's 32-bit sum of d products is off by at most (d + 4) 2^-24 of the
    sum of their sizes, in units of the scaled score; a weight by twice that
    (its own and the maximum's) plus 2^-20 for its exponential and the sums."""
    d = q.shape[-1]
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    g = heads // kv_heads
    out, bound = np.zeros((heads, d)), np.full((heads, d), 2.0 ** -25)
    n = len(k)
    if n == 0:
        return out, bound
    for h in range(heads):
        kh, vh = k[:, h // g], v[:, h // g]
        s = kh @ q[h] / np.sqrt(d)
        p = np.exp(s - s.max())
        w = p / p.sum()
        out[h] = w @ vh
        size = w @ np.abs(vh)
        score = (d + 4) * 2.0 ** -24 * (np.abs(kh) @ np.abs(q[h])).max() / np.sqrt(d)
        bound[h] = (2.0 ** -11 * (1 + 2.0 ** -9) * np.abs(out[h]) + (2.0 ** -11 + 2 * score + 2.0 ** -20) * size +
                    n * 2.0 ** -25 * np.abs(vh).max() / p.sum() + 2.0 ** -25)
    return out, bound


def attend64_wide(q, k, v, heads, kv_heads):
    """attend64 with the bound of kernels that multiply weights of more than 16 bits.

    A weight p is off by 2^-22 of it (two 16-bit numbers: 2^-11 of what the
    first leaves, itself 2^-11 of p) or, where that is more, by 2^-25, the
    largest being at least 2^7: n 2^-32 of the largest |v| in all. Sums of
    products over 16 tokens are added up in 32 bits: 2^-22 of the sum of sizes
    for each of n / 16, and for 64 joins of partial sums. The scores, the
    exponentials and the output's one rounding are as in attend64."""
    d = q.shape[-1]
    out, _ = attend64(q, k, v, heads, kv_heads)
    q, k, v = q.astype(np.float64), k.astype(np.float64), np.abs(v.astype(np.float64))
    size, _ = attend64(q, k, v, heads, kv_heads)
    n, g = len(k), heads // kv_heads
    bound = np.full((heads, d), 2.0 ** -25)
    for h in range(heads) if n else ():
        score = (d + 4) * 2.0 ** -24 * (np.abs(k[:, h // g]) @ np.abs(q[h])).max() / np.sqrt(d)
        bound[h] += (2.0 ** -11 * (1 + 2.0 ** -9) * np.abs(out[h]) + n * 2.0 ** -32 * v[:, h // g].max() +
                     (2 * score + 2.0 ** -20 + (n / 16 + 64 + 1) * 2.0 ** -22) * size[h])
    return out, bound


def assert_within(got, want, bound):
    got = np.asarray(got, np.float64)
    assert np.all(np.isfinite(got))
    over = np.abs(got - want) / bound
    assert over.max() <= 1.0, f"{over.max():.3f} of the bound at {np.unravel_index(over.argmax(), over.shape)}"
