"""The 4-bit key/value cache and the rotation on the way into a cache from
their definitions, in 64 bits on the CPU: test infrastructure only."""
import math
from fractions import Fraction

import numpy as np

from kv_reference import EXP_MAX, EXP_MIN, RefCache

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
SCALES = np.array([n * 2.0 ** k for k in range(-24, 11) for n in range(32, 64)])


def round_e2m1(y):
    """Nearest E2M1 value, ties to the even code, magnitudes past 6 to 6."""
    a = np.minimum(np.abs(y), 6.0)
    d = np.abs(a[..., None] - E2M1)
    low = np.argmin(d, -1)                      # the first of two equally near ones
    high = np.minimum(low + 1, 7)
    tie = np.take_along_axis(d, low[..., None], -1) == np.take_along_axis(d, high[..., None], -1)
    code = np.where(tie[..., 0] & (low % 2 == 1), high, low)
    return np.copysign(E2M1[code], y)


def key_exponent(top):
    e = EXP_MIN
    while e < EXP_MAX and top > 6 * math.ldexp(1.0, e):
        e += 1
    return e


def value_scale(top):
    return SCALES[min(np.searchsorted(6 * SCALES, top), len(SCALES) - 1)]


def encode_keys4(x):
    """Keys [..., dim] as the cache stores them."""
    x = np.asarray(x, np.float64)
    g = x.reshape(-1, 32)
    out = np.full(g.shape, np.nan)
    for i, row in enumerate(g):
        if np.isfinite(row).all():
            power = math.ldexp(1.0, key_exponent(np.abs(row).max()))
            out[i] = round_e2m1(row / power) * power
    return out.reshape(x.shape)


def encode_values4(x):
    x = np.asarray(x, np.float64)
    g = x.reshape(-1, x.shape[-1])
    out = np.full(g.shape, np.nan)
    for i, row in enumerate(g):
        if np.isfinite(row).all():
            s = value_scale(np.abs(row).max())
            out[i] = round_e2m1(row / s) * s
    return out.reshape(x.shape)


class RefCache4(RefCache):
    """Tokens stand alone: an append changes nothing but its own."""

    def append(self, k, v, lengths, tables, counts, weights=None):
        row = 0
        for length, table, n in zip(lengths, tables, counts):
            length = min(max(int(length), 0), len(table) * self.bt)
            for i in range(n):
                t = length - n + i
                b = self.block(table, t // self.bt) if t >= 0 else None
                if b is None:
                    continue
                at = (b, slice(None), t % self.bt)
                self.val[0][at] = encode_keys4(k[row + i])
                self.val[1][at] = encode_values4(v[row + i])
                self.w[at] = 0 if weights is None else weights[row + i]
            row += n

    def attend(self, q, lengths, tables, counts, scale, window=0, accumulate=False):
        """Results as RefCache's, with the bound of this cache's arithmetic: a
        weight times its value's scale is rounded to f16, with 2^-11 of it or, for
        each token seen, 2^-36 of the row's largest such product (times a code of
        6 at most); powers, sums and the quotient in f32 within 2^-17; scores as
        there; the result to bf16."""
        out, _, lse, lse_tol, added_tol = super().attend(q, lengths, tables, counts, scale, window,
                                                         accumulate)
        tol = np.zeros(out.shape)
        group, row = q.shape[1] // self.heads, 0
        for length, table, n in zip(lengths, tables, counts):
            length = min(max(int(length), 0), len(table) * self.bt)
            pos, tok = length - n + np.arange(n)[:, None], np.arange(length)[None]
            for h in range(self.heads if n else 0):
                k, v, _, there = self.tokens(table, length, h)
                see = (tok <= pos) & there[None]
                if window:
                    see = see & (tok > pos - window)
                k, v = np.nan_to_num(k), np.nan_to_num(v)    # rows of NaN have no bound
                each = np.abs(v).max(1) / 4                  # a scale is at most that
                for hh in range(h * group, (h + 1) * group):
                    x = np.nan_to_num(q[row:row + n, hh], posinf=0, neginf=0)
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = np.where(see, scale * (x @ k.T), -np.inf)
                        size = np.abs(x) @ np.abs(k).T * 2.0 ** -20 + \
                            np.max(np.abs(x), 1, initial=0)[:, None] * \
                            np.abs(k).sum(1)[None] * 2.0 ** -22
                        eps = np.max(np.where(see, abs(scale) * size, 0), 1, initial=0)
                        top = np.max(s, 1, initial=-np.inf)
                        p = np.exp(s - np.where(np.isfinite(top), top, 0)[:, None])
                        total = p.sum(1)
                        p = np.where(see, p / np.where(total == 0, 1, total)[:, None], 0)
                    most = np.max(p * each[None], 1, initial=0)
                    part = (2.0 ** -11 + 2.0 ** -17 + 2 * eps)[:, None] * (p @ np.abs(v)) + \
                        2.0 ** -36 * (most * see.sum(1) * 6)[:, None]
                    o = out[row:row + n, hh]
                    tol[row:row + n, hh] = part + 2.0 ** -8 * (np.abs(o) + part)
            row += n
        return out, tol, lse, lse_tol, added_tol

    def evict(self, lengths, tables, new_tables, keep, sink, recent):
        # Codes move as they are: stored values, stored again, are the same.
        return super().evict(lengths, tables, new_tables, keep, sink, recent)


# ------------------------------------------------------------------- rotation

TWO_PI = 2 * Fraction(314159265358979323846264338327950288419716939937510582097494459230781640629,
                      10 ** 74)


def angle(position, freq):
    """position * freq, reduced to -pi .. pi without rounding, then to 64 bits."""
    a = Fraction(int(position)) * Fraction(float(freq))
    return float(a - round(a / TWO_PI) * TWO_PI)


def rotate(x, positions, inv_freq, pair_axes=None, interleaved=False):
    """x float64 [rows][heads][dim], positions [axes][rows], in 64 bits."""
    half = len(inv_freq)
    axes = [0] * half if pair_axes is None else [min(int(a), len(positions) - 1) for a in pair_axes]
    y = np.array(x, np.float64)
    for j in range(half):
        first, second = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        known = {}
        a = np.array([known.setdefault(p, angle(p, inv_freq[j]))
                      for p in np.asarray(positions)[axes[j]].tolist()])[:, None]
        u, w = x[..., first], x[..., second]
        y[..., first] = u * np.cos(a) - w * np.sin(a)
        y[..., second] = w * np.cos(a) + u * np.sin(a)
    return y

