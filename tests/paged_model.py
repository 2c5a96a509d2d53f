"""The paged 8-bit cache's definitions in plain Python and 64-bit numbers: what the CUDA kernels are compared with."""
import math

import numpy as np

FLOOR = -100                      # least exponent of a scale


def exponent(top):
    """The least e >= FLOOR with which top / 2^e rounds to at most 127 (ties to even: 127.5 is 128)."""
    if not np.isfinite(top):
        return None
    e = FLOOR
    if top > 0:
        e = max(e, math.frexp(top)[1] - 8)
    while math.ldexp(top, -e) >= 127.5:
        e += 1
    return e


class Model:
    """One layer.  codes [pages, page, heads, dim] per tensor, exponents [pages, heads] (None: not a number)."""

    def __init__(self, heads, dim, pages, page):
        self.heads, self.dim, self.page = heads, dim, page
        self.stack = list(range(pages))[::-1]
        self.tables, self.lengths, self.batch = {}, {}, []
        self.codes = [np.zeros((pages, page, heads, dim)) for _ in range(2)]
        self.exps = [np.full((pages, heads), FLOOR, object) for _ in range(2)]

    def up(self, n):
        return -(-n // self.page)

    def plan(self, counts, rows=None):
        """[(row, first row of the step, tokens held before, new ones)], slots, positions"""
        rows = range(len(counts)) if rows is None else rows
        self.batch, slots, positions, at = [], [], [], 0
        for r, c in zip(rows, counts):
            table, old = self.tables.setdefault(r, []), self.lengths.get(r, 0)
            while len(table) < self.up(old + c):
                table.append(self.stack.pop())
            self.lengths[r] = old + c
            self.batch.append((r, at, old, c))
            at += c
            for p in range(old, old + c):
                slots.append(table[p // self.page] * self.page + p % self.page)
                positions.append(p)
        return slots, positions

    def truncate(self, lengths, rows=None):
        rows = range(len(lengths)) if rows is None else rows
        freed = []
        for r, n in zip(rows, lengths):
            table = self.tables.setdefault(r, [])
            freed += table[self.up(n):]
            del table[self.up(n):]
            self.lengths[r] = n
        self.stack += freed[::-1]

    def append(self, which, x):
        """x [tokens, heads, dim]"""
        x = np.asarray(x, np.float64)
        for r, at, old, c in self.batch:
            p = old
            while p < old + c:
                page, off = self.tables[r][p // self.page], p % self.page
                n = min(self.page - off, old + c - p)
                new = x[at + p - old:at + p - old + n]
                for h in range(self.heads):
                    before = self.exps[which][page, h] if off else FLOOR
                    mine = exponent(np.abs(new[:, h]).max()) if np.isfinite(new[:, h]).all() else None
                    codes = self.codes[which][page, :, h]
                    if before is None or mine is None:
                        self.exps[which][page, h] = None
                        codes[off:off + n] = 0
                        continue
                    e = max(before, mine)
                    if off and e > before:
                        codes[:off] = np.rint(np.ldexp(codes[:off], before - e))
                    codes[off:off + n] = np.rint(np.ldexp(new[:, h], -e))
                    self.exps[which][page, h] = e
                p += n

    def values(self, which, pages):
        """[n, page, heads, dim]"""
        out = np.empty((len(pages), self.page, self.heads, self.dim))
        for i, p in enumerate(pages):
            for h in range(self.heads):
                e = self.exps[which][p, h]
                out[i, :, h] = np.nan if e is None else np.ldexp(self.codes[which][p, :, h], e)
        return out

    def held(self, which, row):
        """[tokens, heads, dim] of a request"""
        return self.values(which, self.tables[row]).reshape(-1, self.heads, self.dim)[:self.lengths[row]]

    def attention(self, q, window=0, scale=None):
        """q [tokens, q_heads, dim] -> out, lse, and a bound of each element's error: see `bounds`."""
        q = np.asarray(q, np.float64)
        group = q.shape[1] // self.heads
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        out, lse = np.zeros(q.shape), np.zeros(q.shape[:2])
        tol, ltol = np.zeros(q.shape), np.zeros(q.shape[:2])
        for r, at, old, c in self.batch:
            if c == 0:
                continue
            k, v = self.held(0, r), self.held(1, r)
            t = np.arange(old + c)[None]
            p = np.arange(old, old + c)[:, None]
            seen = t <= p
            if window:
                seen &= t > p - window
            for hq in range(q.shape[1]):
                x, kh, vh = q[at:at + c, hq], k[:, hq // group], v[:, hq // group]
                bad = np.isnan(kh).any(1) | np.isnan(vh).any(1)      # tokens of a page and head that is not a number
                kh, vh = np.where(bad[:, None], 0, kh), np.where(bad[:, None], 0, vh)
                s = np.where(seen, x @ kh.T * scale, -np.inf)
                top = s.max(1, keepdims=True)
                w = np.exp(s - top)
                total = w.sum(1, keepdims=True)
                w /= total
                o = w @ vh
                out[at:at + c, hq] = o
                lse[at:at + c, hq] = (top + np.log(total))[:, 0]
                tol[at:at + c, hq], ltol[at:at + c, hq] = bounds(x, kh, vh, w, o, lse[at:at + c, hq], scale, seen)
                lost = (seen & bad[None]).any(1)
                out[at:at + c, hq][lost] = np.nan
                lse[at:at + c, hq][lost] = np.nan
        return out, lse, tol, ltol


def bounds(x, k, v, w, o, lse, scale, seen):
    """How far fp16 results may be off.

    A score is a sum of D exact products, added in fp32 (an addition may lose two units of 2^-24 of the partial sums' magnitude, at
    most sum |q||k|), then two roundings and the exponential's two units: relative error of a weight, against the others,
    a = 2 (D + 8) 2^-24 scale max sum |q||k| + 2^-20.  Weights are rounded to halves: 2^-11 of each.  Small ones are
    subnormal halves, multiples of 2^-24 and so 2^-25 off at most; the kernels hold weights times 2^11 (few rows) or 2^7 (many), against a
    maximum that is no larger than the row's: 2^-25-7 = 2^-32 of the largest weight at most, n 2^-32 max |v| of the sum.  The sums of n terms in fp32: 2 n 2^-24 at worst, of sum w|v|; n 2^-24 for the denominator.
    The result is rounded to a half: 2^-11 of it, or 2^-25 where it is subnormal."""
    d, n = k.shape[1], k.shape[0]
    reach = (np.where(seen, np.abs(x) @ np.abs(k).T, 0)).max(1) * scale
    a = (2 * (d + 8) * 2.0 ** -24 * reach + 2.0 ** -20)[:, None]
    mass = w @ np.abs(v)
    near = np.where(seen[:, :, None], np.abs(v)[None], 0).max((0, 1)) if v.size < 1 << 22 else np.abs(v).max(0)
    before = mass * (2.0 ** -11 + 2 * a + 3 * n * 2.0 ** -24) + n * 2.0 ** -32 * near
    return (np.abs(o) + before) * 2.0 ** -11 + 2.0 ** -25 + before, 2 * a[:, 0] + n * 2.0 ** -24 + 2.0 ** -22 * (np.abs(lse) + 16)
