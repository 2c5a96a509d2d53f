"""A drafted decoding step's definitions in plain Python and 64-bit numbers: what the CUDA kernels are compared with."""
import math

import numpy as np

from tests.paged_model import FLOOR, exponent


def trees(rng, counts, spread):
    """Parents of each request's nodes, a node's among the `spread` in front of it (0: the token in front, a chain)."""
    return [[-1] + [max(0, j - 1 - int(rng.integers(max(1, spread)))) for j in range(1, c)] if c else [] for c in counts]


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def ancestors(parents):
    """[j, i]: i is an ancestor of j, or j."""
    a = np.zeros((len(parents), len(parents)), bool)
    for j, p in enumerate(parents):
        if p >= 0:
            a[j] = a[p]
        a[j, j] = True
    return a


def verify(parents, tokens, target, draft, u, width):
    """One request: rows of target and draft (None) by node -> path, next token."""
    clean = lambda x: np.where(x > 0, np.asarray(x, np.float64), 0)                    # noqa: E731
    if not len(parents):
        return [], -1
    vocab, now, path = target.shape[1], 0, [0]
    w, z = clean(target[0]), 1.0
    q = None if draft is None else clean(draft[0])
    for c in range(1, min(len(parents), 1024)):
        x = tokens[c]
        if len(path) == width or parents[c] != now or not 0 <= parents[c] < c or not 0 <= x < vocab:
            continue
        if float(u[c]) * z * (1.0 if q is None else q[x]) < w[x]:
            now = c
            path.append(c)
            w, z = clean(target[c]), 1.0
            q = None if draft is None else clean(draft[c])
        elif q is None:
            z -= w[x]
            w[x] = 0
        else:
            w = np.maximum(w - z * q, 0)
            z = w.sum()
    if not w.sum() > 0:
        w = clean(target[now])
    if not w.sum() > 0:
        return path, -1
    sums = np.cumsum(w)
    beyond = np.nonzero((sums > float(u[0]) * sums[-1]) & (w > 0))[0]
    return path, int(beyond[0] if len(beyond) else np.nonzero(w > 0)[0][-1])


def keep(m, which, paths):
    """Codes and scales of a paged_model.Model's last plan, keys or values, when the tokens of `paths` have moved up (None: all stay)."""
    for (r, _, old, _), path in zip(m.batch, paths):
        if path is None:
            continue
        table = m.tables[r]
        for page in range(old // m.page, (old + max(len(path), 1) - 1) // m.page + 1):
            mine = [(old + a, old + i) for i, a in enumerate(path) if (old + i) // m.page == page and a != i]
            for h in range(m.heads):
                codes, exps = m.codes[which][:, :, h], m.exps[which][:, h]
                here = table[page] if page < len(table) else None
                others = []
                for a, i in mine:
                    if a // m.page == page:
                        codes[here, i % m.page] = codes[here, a % m.page]
                    else:
                        others.append((table[a // m.page], a % m.page, i % m.page))
                if not others:
                    continue
                if exps[here] is None or any(exps[p] is None for p, _, _ in others):
                    exps[here] = None
                    for _, _, i in others:
                        codes[here, i] = 0
                    continue
                moved = [(i, np.ldexp(codes[p, a], exps[p])) for p, a, i in others]
                e = max(exps[here], max(exponent(np.abs(v).max()) for _, v in moved), FLOOR)
                codes[here] = np.rint(np.ldexp(codes[here], exps[here] - e))
                exps[here] = e
                for i, v in moved:
                    codes[here, i] = np.rint(np.ldexp(v, -e))


def kept_lengths(m, paths):
    return [old + (c if path is None else len(path)) for (_, _, old, c), path in zip(m.batch, paths)]


def qk_norm_rope(x, w, positions, theta, eps):
    """x [tokens, heads, dim] -> the result and a bound of each fp16 result's error.

    The sum of D squares in fp32 is D 2^-24 off at most (relative), its root's inverse half of that and two units; the products with it
    and the weight, a unit each.  Sine and cosine are two units of 2^-24 off, and their angle, a multiple of 2^-31 half turns below 1
    rounded to 24 bits, pi 2^-24.  So each product of the rotation is (D / 2 + 16) 2^-24 of itself off, and the sum one unit more; the
    result is rounded to a half: 2^-11 of it, or 2^-25 where it is subnormal."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    dim = x.shape[2]
    with np.errstate(all="ignore"):
        y = x / np.sqrt((x ** 2).mean(2, keepdims=True) + eps) * w
        angle = np.asarray(positions, np.float64)[:, None, None] * theta ** (-2 * np.arange(dim // 2) / dim)
        c, s, a, b = np.cos(angle), np.sin(angle), y[..., :dim // 2], y[..., dim // 2:]
        want = np.concatenate([a * c - b * s, b * c + a * s], 2)
        off = np.concatenate([np.abs(a) + np.abs(b)] * 2, 2) * (dim / 2 + 17) * 2.0 ** -24
    return want, (np.abs(want) + off) * 2.0 ** -11 + 2.0 ** -25 + off
