"""Attention over the paged cache in 64-bit numbers, with a bound of each result's error that knows what each row sees and which
kernel its request takes."""
import math

import numpy as np

FEW_ROWS = 16      # query rows of a request up to which the kernel for few rows takes it
LOST = 30          # a page's numbers are 0 for many rows where its scale is 2^-30 of its 64 tokens' largest, or less


def held(model, which, row, head, many):
    """A request's values as the kernel has them [tokens, dim], and 127 times each token's scale."""
    pages = model.tables[row]
    e = [model.exps[which][p, head] for p in pages]
    at_once = max(1, 64 // model.page)
    out, most = np.empty((len(pages), model.page, model.dim)), np.empty((len(pages), model.page))
    for i, p in enumerate(pages):
        largest = max(e[i // at_once * at_once:(i // at_once + 1) * at_once])
        gone = many and e[i] <= largest - LOST
        out[i] = 0 if gone else np.ldexp(model.codes[which][p, :, head], e[i])
        most[i] = math.ldexp(127, e[i])
    n = model.lengths[row]
    return out.reshape(-1, model.dim)[:n], most.reshape(-1)[:n]


def attention(model, q, window=0):
    """q [tokens, q_heads, dim] -> out, lse, tol, ltol; pages are numbers.

    As paged_model.bounds has it, but for the weights: held times 2^11 (few rows) or 2^7 (many) as halves, and multiplied with a page's
    scale against the largest that the row has met, they are off by 2^-25-11 or 2^-25-7 of the largest weight times the largest of
    127 times the scales that the row sees, n times in the sum.  What a row does not see is in none of its bounds."""
    q = np.asarray(q, np.float64)
    group, dim = q.shape[1] // model.heads, model.dim
    scale = 1 / math.sqrt(dim)
    out, lse = np.zeros(q.shape), np.zeros(q.shape[:2])
    tol, ltol = np.zeros(q.shape), np.zeros(q.shape[:2])
    for r, at, old, c in model.batch:
        if c == 0:
            continue
        many = c * group > FEW_ROWS
        t, p = np.arange(old + c)[None], np.arange(old, old + c)[:, None]
        seen = (t <= p) & ((t > p - window) if window else True)
        n = seen.sum(1)
        for head in range(model.heads):
            (k, _), (v, most) = (held(model, which, r, head, many) for which in (0, 1))
            near = np.where(seen, most[None], 0).max(1)
            for hq in range(head * group, (head + 1) * group):
                x = q[at:at + c, hq]
                s = np.where(seen, x @ k.T * scale, -np.inf)
                top = s.max(1, keepdims=True)
                w = np.where(seen, np.exp(s - top), 0)
                total = w.sum(1, keepdims=True)
                w /= total
                o, mass = w @ v, w @ np.abs(v)
                reach = np.where(seen, np.abs(x) @ np.abs(k).T, 0).max(1) * scale
                a = 2 * (dim + 8) * 2.0 ** -24 * reach + 2.0 ** -20
                before = mass * (2.0 ** -11 + 2 * a + 3 * n * 2.0 ** -24)[:, None] + (n * 2.0 ** (-32 if many else -36) * near)[:, None]
                out[at:at + c, hq] = o
                lse[at:at + c, hq] = (top + np.log(total))[:, 0]
                tol[at:at + c, hq] = (np.abs(o) + before) * 2.0 ** -11 + 2.0 ** -25 + before
                ltol[at:at + c, hq] = 2 * a + n * 2.0 ** -24 + 2.0 ** -22 * (np.abs(lse[at:at + c, hq]) + 16)
    return out, lse, tol, ltol
