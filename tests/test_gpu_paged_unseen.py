"""GPU tests of attention where the tokens that a row does not see have scales far from those that it sees, with bounds that go by each
row's own tokens."""
import numpy as np
import pytest

from tests.paged_bounds import attention
from tests.paged_model import Model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def compare(got, lse, want):
    out, sums, tol, ltol = want
    got, lse = got.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    with np.errstate(over="ignore"):
        large = ~np.isfinite(out.astype(np.float16)) | (np.abs(out) > 60000)     # (rows that see the large value)
    assert np.isfinite(got[~large]).all()
    worst = np.max((np.abs(got - out) / tol)[~large], initial=0)
    assert worst <= 1, f"outputs off by {worst} times their bound"
    worst = np.max(np.abs(lse - sums) / ltol)
    assert worst <= 1, f"log sums off by {worst} times their bound"
    return large


def run(c, q, **more):
    lse = torch.full(q.shape[:2], 9.0, device="cuda")
    out = c.attention(0, q, out=torch.full_like(q, 9.0), lse=lse, **more)
    torch.cuda.synchronize()
    c.check_status()
    return out, lse


def served(tq, rng, heads, dim, page, prompts, last, change, times=1):
    """A cache and its model after prompts and then the tokens `last`; change(k, v, i) alters request i's tokens.  `times`: the cache holds all of it
    so many times, one behind the other, the model once."""
    total = [a + b for a, b in zip(prompts, last)]
    need = [-(-t // page) for t in total]
    c = tq.PagedKVCache(1, heads, dim, times * sum(need), page, times * len(total), max(need), times * max(sum(prompts), sum(last)))
    m = Model(heads, dim, sum(need), page)
    data = []
    for i, t in enumerate(total):
        k, v = (rng.standard_normal((t, heads, dim)).astype(np.float32) for _ in range(2))
        change(k, v, i)
        data.append((k, v))
    for counts, part in ((prompts, [(0, p) for p in prompts]), (last, [(p, t) for p, t in zip(prompts, total)])):
        m.plan(counts)
        c.plan(np.array(times * counts, np.int32))
        k, v = (np.concatenate([data[i][which][a:b] for i, (a, b) in enumerate(part)]) for which in (0, 1))
        m.append(0, k)
        m.append(1, v)
        c.append(0, *(torch.from_numpy(x).cuda().repeat(times, 1, 1) for x in (k, v)))
    return c, m


def queries(rng, tokens, q_heads, dim):
    return rng.standard_normal((tokens, q_heads, dim)).astype(np.float16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page,edge", [(16, 96), (32, 96), (64, 128), (128, 128)])
@pytest.mark.parametrize("group,last", [(1, 2), (4, 2), (8, 2), (1, 9), (5, 3), (1, 16)])
@pytest.mark.parametrize("large", [2.0 ** 20, 2.0 ** 32, 1e15])
def test_a_window_that_ends_between_few_rows(tq, dim, page, edge, group, last, large):
    """The first draft sees a large value, the last token of its page, and the ones behind it do not: these go by their own scales.  (So many
    requests that a CTA goes through several tiles of one.)"""
    rng = np.random.default_rng(dim + page + last)
    requests = 160

    def change(k, v, i):
        v[edge - 1] = large
        k[edge - 1] = 0
    c, m = served(tq, rng, 4, dim, page, [edge + 165], [last], change, requests)
    q = queries(rng, last, 4 * group, dim)
    # row 0 at position edge + 165 sees from edge - 1 on
    out, lse = run(c, torch.from_numpy(q).cuda().repeat(requests, 1, 1), window=167)
    want = attention(m, q, 167)
    for o, l in zip(out.split(last), lse.split(last)):
        assert not compare(o, l, want)[1:].any()
    c.close()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,last", [(1, 1), (2, 8), (7, 1), (16, 1), (1, 16), (3, 3)])
@pytest.mark.parametrize("window", [0, 50])
def test_few_rows_within_their_own_bound(tq, dim, group, last, window):
    """Scales that change from page to page by up to 2^12, in every order, and drafts of which the later ones are large."""
    rng = np.random.default_rng(dim + group)
    lift = np.exp2(rng.integers(0, 13, 400))

    def change(k, v, i):
        v *= lift[np.arange(len(v)) // 16, None, None].astype(np.float32)
        v[-1] = 1e15 if i % 2 else v[-1]
        k *= np.exp2(rng.integers(-3, 3, (len(k), 1, 1))).astype(np.float32)
    c, m = served(tq, rng, 2, dim, 16, [700, 45, 333, 1], [last] * 4, change)
    q = queries(rng, 4 * last, 2 * group, dim)
    compare(*run(c, torch.from_numpy(q).cuda(), window=window), attention(m, q, window))
    c.close()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("group,last,window", [(1, 60, 100), (7, 30, 100), (2, 200, 130), (1, 300, 257)])
@pytest.mark.parametrize("large", [2.0 ** 20, 2.0 ** 27, 1e15])
def test_a_window_that_ends_inside_a_tile_of_many_rows(tq, dim, page, group, last, window, large):
    """A value is large at the beginning of 64 tokens, and windows begin there, behind it in its page and in the pages behind: a row goes by the
    scales that it sees, in these 64 tokens and in the ones behind them."""
    rng = np.random.default_rng(dim + page + last)
    requests, edge = 25, 128

    def change(k, v, i):
        v[edge] = large
        k[edge] = 0
    # row 0 sees from edge - 3 on
    c, m = served(tq, rng, 4, dim, page, [edge + window - 4], [last], change, requests)
    q = queries(rng, last, 4 * group, dim)
    out, lse = run(c, torch.from_numpy(q).cuda().repeat(requests, 1, 1), window=window)
    want = attention(m, q, window)
    for o, l in zip(out.split(last), lse.split(last)):
        assert not compare(o, l, want)[4:].any()
    c.close()
