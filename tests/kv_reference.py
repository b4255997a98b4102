"""The key/value cache and its attention from their definitions, in 64 bits on
the CPU: test infrastructure only.  Values are held as float64, exponents as
integers; every operation is written out per sequence, head and block."""
import math

import numpy as np

EXP_MIN, EXP_MAX = -100, 119


def exponent(values):
    """Smallest e with |finite values| <= 448 * 2^e, clamped."""
    a = np.abs(values[np.isfinite(values)])
    top = float(a.max()) if a.size else 0.0
    e = EXP_MIN
    while e < EXP_MAX and top > 448.0 * math.ldexp(1.0, e):
        e += 1
    return e


def encode(values, e):
    """Values rounded to E4M3 multiples of 2^e (ties to even), saturated;
    infinities and NaN become NaN."""
    x, e = np.asarray(values, np.float64), int(e)
    y = np.abs(np.where(np.isfinite(x), x, 0.0)) * math.ldexp(1.0, -e)
    _, ex = np.frexp(np.maximum(y, 2.0 ** -6))
    q = np.ldexp(1.0, ex - 4)
    r = np.minimum(np.round(y / q) * q, 448.0) * math.ldexp(1.0, e)
    return np.where(np.isfinite(x), np.copysign(r, x), np.nan)


class RefCache:
    def __init__(self, blocks, heads, dim, bt):
        self.blocks, self.heads, self.dim, self.bt = blocks, heads, dim, bt
        self.val = np.zeros((2, blocks, heads, bt, dim))
        self.exp = np.zeros((2, blocks, heads), int)
        self.w = np.zeros((blocks, heads, bt))

    def block(self, table, j):
        if j >= len(table) or not 0 <= table[j] < self.blocks:
            return None
        return int(table[j])

    def append(self, k, v, lengths, tables, counts, weights=None):
        """k, v float64 [rows][heads][dim]; counts: rows of each sequence."""
        row = 0
        for length, table, n in zip(lengths, tables, counts):
            length = min(max(int(length), 0), len(table) * self.bt)
            origin = length - n
            for j in range(max(origin, 0) // self.bt, -(-length // self.bt) if n else 0):
                lo, hi = max(origin, j * self.bt, 0), min(length, (j + 1) * self.bt)
                b = self.block(table, j)
                if b is None or lo >= hi:
                    continue
                rows = slice(row + lo - origin, row + hi - origin)
                at = slice(lo - j * self.bt, hi - j * self.bt)
                for side, x in enumerate((k, v)):
                    for h in range(self.heads):
                        e = exponent(x[rows, h])
                        if at.start > 0:
                            e = max(e, self.exp[side, b, h])
                            old = self.val[side, b, h, :at.start]
                            self.val[side, b, h, :at.start] = encode(old, e)
                        self.exp[side, b, h] = e
                        self.val[side, b, h, at] = encode(x[rows, h], e)
                self.w[b, :, at] = 0 if weights is None else weights[rows].T
            row += n

    def tokens(self, table, length, h):
        """(k, v [length][dim], weights, present) of a head's tokens."""
        k, v = np.zeros((length, self.dim)), np.zeros((length, self.dim))
        w, there = np.zeros(length), np.zeros(length, bool)
        for t in range(length):
            b = self.block(table, t // self.bt)
            if b is not None:
                k[t], v[t] = self.val[:, b, h, t % self.bt]
                w[t], there[t] = self.w[b, h, t % self.bt], True
        return k, v, w, there

    def gather(self, lengths, tables, counts):
        rows = sum(counts)
        k, v = np.zeros((2, rows, self.heads, self.dim))
        w = np.zeros((rows, self.heads))
        row = 0
        for length, table, n in zip(lengths, tables, counts):
            length = min(max(int(length), 0), len(table) * self.bt)
            for h in range(self.heads):
                kk, vv, ww, _ = self.tokens(table, length, h)
                m = min(n, length)
                k[row + n - m:row + n, h] = kk[length - m:]
                v[row + n - m:row + n, h] = vv[length - m:]
                w[row + n - m:row + n, h] = ww[length - m:]
            row += n
        return k, v, w

    def attend(self, q, lengths, tables, counts, scale, window=0, accumulate=False):
        """q float64 [rows][heads][dim].  Returns out, lse and, for each, a bound
        of the error that the documented arithmetic may make (bf16 weights and
        output, f32 scores and sums); `added` is what accumulate adds to self.w,
        with its bound."""
        rows, hq, _ = q.shape
        group = hq // self.heads
        out, out_tol = np.zeros(q.shape), np.zeros(q.shape)
        lse, lse_tol = np.full((rows, hq), -np.inf), np.zeros((rows, hq))
        added, added_tol = np.zeros_like(self.w), np.zeros_like(self.w)
        row = 0
        for length, table, n in zip(lengths, tables, counts):
            length = min(max(int(length), 0), len(table) * self.bt)
            pos = length - n + np.arange(n)[:, None]
            tok = np.arange(length)[None]
            for h in range(self.heads if n else 0):
                k, v, _, there = self.tokens(table, length, h)
                see = (tok <= pos) & there[None]
                if window:
                    see = see & (tok > pos - window)
                for hh in range(h * group, (h + 1) * group):
                    x = q[row:row + n, hh]
                    x = np.where(np.isinf(x), np.nan, x)  # scores of both signs: NaN rows
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = np.where(see, scale * (x @ k.T), -np.inf)
                        # Score error: f32 products and sums, and 2^-22 of the
                        # row's largest element in each element of q.
                        size = np.abs(x) @ np.abs(k).T * 2.0 ** -20 + \
                            np.max(np.abs(x), 1, initial=0)[:, None] * \
                            np.abs(k).sum(1)[None] * 2.0 ** -22
                        eps = np.max(np.where(see, abs(scale) * size, 0), 1, initial=0)
                        top = np.max(s, 1, initial=-np.inf)
                        p = np.exp(s - np.where(np.isfinite(top) | np.isnan(top), top, 0)[:, None])
                        total = p.sum(1)
                        p = np.where(see, p / np.where(total == 0, 1, total)[:, None], 0)
                        if np.isfinite(v).all():
                            o, size = p @ v, p @ np.abs(v)
                        else:  # hidden values take no part, not even as 0 * NaN
                            vv = np.where(see[:, :, None], v[None], 0)
                            o = (p[:, :, None] * vv).sum(1)
                            size = (p[:, :, None] * np.abs(vv)).sum(1)
                        one = np.where(total == 0, -np.inf, np.log(np.maximum(total, 1e-300)) + top)
                    part = (2.0 ** -9 + 2.0 ** -17 + 2 * eps)[:, None] * size
                    out[row:row + n, hh] = o
                    out_tol[row:row + n, hh] = part + 2.0 ** -8 * (np.abs(o) + part)
                    lse[row:row + n, hh] = one
                    lse_tol[row:row + n, hh] = eps + 2.0 ** -20 * np.maximum(
                        1, np.where(np.isfinite(one), np.abs(one), 0))
                    size = (p * (2 * eps + 2.0 ** -18)[:, None]).sum(0)
                    for j in range(-(-length // self.bt)):
                        b, at = self.block(table, j), slice(j * self.bt, (j + 1) * self.bt)
                        if b is not None:
                            m = len(size[at])
                            added[b, h, :m] += p[:, at].sum(0)
                            added_tol[b, h, :m] += size[at]
            row += n
        if accumulate:
            self.w = self.w + added
            added_tol = added_tol + np.abs(self.w) * 2.0 ** -22
        return out, out_tol, lse, lse_tol, added_tol

    def evict(self, lengths, tables, new_tables, keep, sink, recent):
        kept = np.full((len(lengths), self.heads, keep), -1)
        new = []
        for b, (length, table) in enumerate(zip(lengths, tables)):
            length = min(max(int(length), 0), len(table) * self.bt)
            m = min(length, keep)
            new.append(m)
            ks, vs, ws = np.zeros((3, m, self.heads, self.dim))
            for h in range(self.heads):
                k, v, w, there = self.tokens(table, length, h)
                free = range(sink, length - recent) if length > keep else range(0)
                big = np.where(np.isnan(w), np.inf, w)

                def order(t):  # NaN, then the largest, then the lowest position
                    return (not (there[t] and math.isnan(w[t])), -big[t] if there[t] else np.inf, t)
                most = sorted(free, key=order)[:max(m - sink - recent, 0)]
                at = sorted(set(most) | (set(range(length)) - set(free)))
                kept[b, h, :m] = at
                ks[:, h], vs[:, h], ws[:, h, 0] = k[at], v[at], w[at]
            self.append(ks, vs, [m], [new_tables[b]], [m], ws[:, :, 0])
        return kept, new
