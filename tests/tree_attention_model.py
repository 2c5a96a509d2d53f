"""Attention of trees of drafts over a paged_model.Model in 64-bit numbers, with a bound of each result's error."""
import math

import numpy as np

from tests.drafts_model import ancestors, depths

def attention(model, q, parents, window=0, scale=None):
    """q [tokens, q_heads, dim], the last plan's parents -> out, lse, tol, ltol.

    A score is a sum of D exact products in fp32 (2 units of 2^-24 of sum |q||k| for each addition), then scaled, added to the
    value's exponent and taken off a reference: three roundings of at most 2^-24 of the largest of them in powers of two, |s| log2(e) + 130
    + |reference|; with the exponential's two units a weight's relative error is a = 2 (D + 8) 2^-24 scale sum |q||k| + 3 2^-24 (2 |s| log2(e)
    + 260) + 2^-22 (against each other, of two weights twice that).

    Weights are rounded to halves, 2^-11 of each, and subnormal ones to multiples of 2^-24, 2^-25 off.  They are held times 2^7, against a
    maximum that is no larger than the row's, and times a value's scale against the largest that the row has met: a small one's error is 2^-32 of the
    row's largest weight, times 127 times the largest scale that the row sees; n of them.  Sums of n terms in fp32: 2 n 2^-24 of sum w|v|, n 2^-24
    for the denominator; the two halves of a row that two teams have summed are added with two more roundings.  The result is rounded to a half: 2^-11
    of it, or 2^-25 where it is subnormal."""
    q = np.asarray(q, np.float64)
    group, dim = q.shape[1] // model.heads, model.dim
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, lse = np.zeros(q.shape), np.zeros(q.shape[:2])
    tol, ltol = np.zeros(q.shape), np.zeros(q.shape[:2])
    for (r, at, old, c), par in zip(model.batch, parents):
        if c == 0:
            continue
        pages = model.tables[r]
        n = model.lengths[r]
        depth = np.array(depths(par))
        place = np.concatenate([np.arange(old), old + depth])
        seen = np.concatenate([np.ones((c, old), bool), ancestors(par)], 1)
        if window:
            seen &= place[None] > (old + depth - window)[:, None]
        for head in range(model.heads):
            k, v = (model.held(which, r)[:, head] for which in (0, 1))
            exps = [[np.nan if model.exps[which][p, head] is None else model.exps[which][p, head] for p in pages] for which in (0, 1)]
            unit = np.ldexp(1.0, np.nan_to_num(np.repeat(exps[1], model.page)[:n], nan=0).astype(int))      # of each token's values
            bad = np.isnan(k).any(1) | np.isnan(v).any(1)
            k, v = np.where(bad[:, None], 0, k), np.where(bad[:, None], 0, v)
            lost = (seen & bad[None]).any(1)
            for hq in range(head * group, (head + 1) * group):
                x = q[at:at + c, hq]
                s = np.where(seen, x @ k.T * scale, -np.inf)
                top = s.max(1, keepdims=True)
                w = np.where(seen, np.exp(s - top), 0)
                total = w.sum(1, keepdims=True)
                w /= total
                o, mass = w @ v, w @ np.abs(v)
                reach = np.where(seen, np.abs(x) @ np.abs(k).T, 0).max(1) * scale
                far = np.where(seen, np.abs(s, where=seen, out=np.zeros(s.shape)), 0).max(1) * 1.4427
                a = 2 * (dim + 8) * 2.0 ** -24 * reach + 3 * 2.0 ** -24 * (2 * far + 260) + 2.0 ** -22
                most = np.where(seen, unit[None], 0).max(1)
                count = seen.sum(1)
                before = mass * (2.0 ** -11 + 2 * a + (3 * count + 2) * 2.0 ** -24)[:, None] + (count * 2.0 ** -32 * most * 127)[:, None]
                out[at:at + c, hq], lse[at:at + c, hq] = o, (top + np.log(total))[:, 0]
                tol[at:at + c, hq] = (np.abs(o) + before) * 2.0 ** -11 + 2.0 ** -25 + before
                ltol[at:at + c, hq] = 2 * a + count * 2.0 ** -24 + 2.0 ** -22 * (np.abs(lse[at:at + c, hq]) + 100)
                out[at:at + c, hq][lost], lse[at:at + c, hq][lost] = np.nan, np.nan
    return out, lse, tol, ltol
