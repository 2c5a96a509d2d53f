"""GPU tests of pages that hold nothing but what a kept branch brings: drafts that were not numbers and did not stay leave nothing behind."""
import numpy as np
import pytest

from tests.paged_model import FLOOR, exponent
from tests.test_gpu_drafts_cache import Pair, ints, paths_tensor

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def keep(m, which, paths):
    """As drafts_model.keep, and a page that is not a number, of which no token stays, takes its scale from those that join it."""
    for (r, _, old, _), path in zip(m.batch, paths):
        table = m.tables[r]
        for i in range(0, len(path)):
            if i and (old + i) % m.page:
                continue
            place = (old + i) // m.page          # a page, from the path's i-th token on
            mine = [(old + a, old + j) for j, a in enumerate(path) if (old + j) // m.page == place]
            inside = [x for x in mine if x[0] // m.page == place]
            others = [(table[a // m.page], a % m.page, j % m.page) for a, j in mine if a // m.page != place]
            here, empty = table[place], (old + i) % m.page == 0 and not inside
            for h in range(m.heads):
                codes, exps = m.codes[which][:, :, h], m.exps[which][:, h]
                for a, j in inside:
                    codes[here, j % m.page] = codes[here, a % m.page]
                if not others:
                    continue
                if empty and exps[here] is None:
                    exps[here] = FLOOR
                if exps[here] is None or any(exps[p] is None for p, _, _ in others):
                    exps[here] = None
                    for _, _, j in others:
                        codes[here, j] = 0
                    continue
                moved = [(j, np.ldexp(codes[p, a], exps[p])) for p, a, j in others]
                e = max(exps[here], max(exponent(np.abs(v).max()) for _, v in moved))
                codes[here] = np.rint(np.ldexp(codes[here], exps[here] - e))
                exps[here] = e
                for j, v in moved:
                    codes[here, j] = np.rint(np.ldexp(v, -e))


def kept(p, paths, rows):
    p.c.keep(paths_tensor(paths, max(map(len, paths))), ints([len(x) for x in paths]))
    for m in p.m:
        for which in (0, 1):
            keep(m, which, paths)
        m.truncate([old + len(x) for (_, _, old, _), x in zip(m.batch, paths)], rows)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("page,dim", [(16, 64), (16, 128), (32, 64), (64, 128)])
def test_drafts_that_are_not_numbers_and_do_not_stay(tq, bad, page, dim):
    rng = np.random.default_rng(page + dim)
    heads, rows, pages = 2, [0, 1, 2, 3], 60
    p = Pair(tq, heads, dim, page, 4, pages)
    p.step(rng, [page, 0, 2 * page, 3], rows)
    counts, at = [3 * page + 5] * 4, 3 * page + 5
    keys = rng.standard_normal((4 * at, heads, dim)).astype(np.float16)
    keys[3, 0, 5] = keys[page - 1, 1, 0] = bad                        # request 0: its first new page, in both heads
    keys[at + page + 1, 0, 9] = keys[at + 2, 1, 1] = bad              # 1: the second one in a head, the first in the other
    keys[2 * at + 1, 0, 0] = keys[2 * at + page, 0, 0] = bad          # 2: the first two
    keys[3 * at + 4, 0, 7] = bad                                      # 3: a page that holds older tokens
    p.step(rng, counts, rows, keys=keys)
    far = 2 * page + 1
    kept(p, [[page + 1, page + 4, 2 * page, far], [*range(page), 2 * page + 1, 3 * page], [*range(page, 2 * page), far, 3 * page + 4], [far, far + 2]], rows)
    p.compare(pages)
    scales = [p.m[0].exps[0][p.m[0].tables[r][i], :].tolist() for r, i in ((0, 1), (1, 0), (1, 1), (2, 2), (2, 3), (3, 0))]
    assert None not in scales[0] and scales[1][0] is not None and scales[1][1] is None and None not in scales[2]
    assert scales[3][0] is None and scales[3][1] is not None and None not in scales[4] and scales[5][0] is None
    # what comes behind joins at those scales, and request 0 is a request of numbers
    p.step(rng, [5, 1, 3, 0], rows)
    p.compare(pages)
    q = torch.from_numpy(rng.standard_normal((9, heads, dim)).astype(np.float16)).cuda()
    out = p.c.attention(0, q)
    assert torch.isfinite(out[:5]).all() and torch.isnan(out[6:, 0]).all() and torch.isfinite(out[6:, 1]).all()
    p.c.close()


@pytest.mark.parametrize("page", [16, 64])
def test_large_drafts_that_do_not_stay(tq, page):
    """A finite scale stays, whoever raised it: tokens that join are rounded at it."""
    rng = np.random.default_rng(page)
    p = Pair(tq, 1, 64, page, 1, 20)
    p.step(rng, [page], [0])
    keys = rng.standard_normal((2 * page, 1, 64)).astype(np.float16)
    keys[0] = 60000
    p.step(rng, [2 * page], [0], keys=keys)
    kept(p, [[page + 2, page + 3]], [0])
    p.compare(20)
    assert p.m[0].exps[0][p.m[0].tables[0][1], 0] == 9
    p.c.close()


@pytest.mark.parametrize("which", [0, 1])
def test_keys_and_values_each_for_themselves(tq, which):
    """Of fp32 tensors, where either may be out of a half's range."""
    rng = np.random.default_rng(which)
    p = Pair(tq, 2, 64, 16, 2, 30)
    p.step(rng, [16, 3], [0, 1])
    for m in p.m:
        m.plan([40, 40], [0, 1])
    p.c.plan(np.array([40, 40], np.int32), rows=ints([0, 1]))
    kv = [rng.standard_normal((80, 2, 64)).astype(np.float32) for _ in range(2)]
    kv[which][2, 0, 1], kv[which][41 + 13, 1, 63], kv[1 - which][9, 1, 0] = np.inf, np.nan, 3e38
    for i, x in enumerate(kv):
        p.m[0].append(i, x)
    p.c.append(0, *(torch.from_numpy(x).cuda() for x in kv))
    kept(p, [[17, 20, 39], [*range(13), 29, 30]], [0, 1])
    p.compare(30)
    exps = [p.m[0].exps[i][p.m[0].tables[r][1]].tolist() for r in (0, 1) for i in (which, 1 - which)]
    assert None not in exps[0] + exps[1] + exps[2] + exps[3] and exps[1][1] > 100 > exps[0][0]
    p.c.close()
