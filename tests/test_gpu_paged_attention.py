"""GPU tests of attention over the paged cache against its definition in 64 bits, within bounds that follow from the roundings."""
import numpy as np
import pytest

from tests.paged_model import Model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def filled(tq, rng, heads, dim, page, rounds, spread=1.0, max_tokens=None, later=()):
    """A cache and its model after the plans and appends of `rounds`, with room for `later` ones; the last plan is in force."""
    n = len(rounds[0])
    lengths = [sum(r[i] for r in (*rounds, *later)) for i in range(n)]
    need = [-(-a // page) for a in lengths]
    c = tq.PagedKVCache(1, heads, dim, sum(need) + 3, page, n, max(need), max_tokens or max(sum(r) for r in (*rounds, *later)) + 8)
    m = Model(heads, dim, sum(need) + 3, page)
    rows = rng.permutation(n).tolist()
    for counts in rounds:
        m.plan(counts, rows)
        c.plan(np.array(counts, np.int32), rows=ints(rows))
        for which in (0, 1):
            x = (rng.standard_normal((sum(counts), heads, dim)) * np.exp(spread * rng.standard_normal((sum(counts), 1, 1)))).astype(np.float16)
            m.append(which, x)
            if which == 0:
                k = x
        if sum(counts):
            c.append(0, torch.from_numpy(k).cuda(), torch.from_numpy(x).cuda())
    return c, m, rows


def compare(got, lse, want):
    out, sums, tol, ltol = want
    got, lse = got.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(out)) and np.array_equal(np.isnan(lse), np.isnan(sums))
    fine = ~np.isnan(out)
    worst = np.max(np.abs(got - out)[fine] / tol[fine], initial=0)
    assert worst <= 1, f"outputs off by {worst} times their bound"
    fine = ~np.isnan(sums)
    worst = np.max(np.abs(lse - sums)[fine] / ltol[fine], initial=0)
    assert worst <= 1, f"log sums off by {worst} times their bound"


def run(c, q, **more):
    lse = torch.full(q.shape[:2], 9.0, device="cuda")
    out = c.attention(0, q, out=torch.full_like(q, 9.0), lse=lse, **more)
    torch.cuda.synchronize()
    c.check_status()
    return out, lse


def queries(rng, tokens, q_heads, dim):
    return (1.5 * rng.standard_normal((tokens, q_heads, dim))).astype(np.float16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 7), (3, 5), (1, 16), (2, 24)])
def test_single_tokens(tq, dim, page, heads, group):
    rng = np.random.default_rng(dim + page + group)
    held = [0, 1, 15, 16, 63, 64, 127, 200, 333]
    c, m, _ = filled(tq, rng, heads, dim, page, [held, [1] * len(held)])
    q = queries(rng, len(held), heads * group, dim)
    compare(*run(c, torch.from_numpy(q).cuda()), m.attention(q))
    c.close()


@pytest.mark.parametrize("dim,page,heads,group", [(128, 64, 2, 7), (128, 16, 1, 8), (64, 32, 2, 4), (128, 128, 1, 1), (64, 64, 1, 40)])
@pytest.mark.parametrize("rounds", [
    [[1]], [[2]], [[5, 0, 3]], [[17, 129, 1]], [[100], [7]], [[0, 300, 64], [1, 4, 130]], [[130, 70], [257, 1]], [[40] * 20, [3] * 20], [[513]]])
def test_prompts_chunks_and_drafts(tq, dim, page, heads, group, rounds):
    rng = np.random.default_rng(dim + group)
    c, m, _ = filled(tq, rng, heads, dim, page, rounds)
    q = queries(rng, sum(rounds[-1]), heads * group, dim)
    compare(*run(c, torch.from_numpy(q).cuda()), m.attention(q))
    c.close()


@pytest.mark.parametrize("dim,page", [(128, 16), (64, 128)])
@pytest.mark.parametrize("window", [1, 2, 15, 64, 65, 200, 5000])
@pytest.mark.parametrize("rounds", [[[300, 64, 1], [1, 1, 1]], [[260, 0], [70, 130]], [[500], [6]]])
def test_windows(tq, dim, page, window, rounds):
    rng = np.random.default_rng(window)
    c, m, _ = filled(tq, rng, 2, dim, page, rounds)
    q = queries(rng, sum(rounds[-1]), 6, dim)
    compare(*run(c, torch.from_numpy(q).cuda(), window=window), m.attention(q, window))
    c.close()


@pytest.mark.parametrize("rounds", [[[40000, 3], [1, 1]], [[2500] * 40, [1] * 40], [[9000], [40]]])
def test_items_that_many_ctas_share(tq, rounds):
    rng = np.random.default_rng(5)
    c, m, _ = filled(tq, rng, 1, 128, 64, rounds, max_tokens=100008)
    q = queries(rng, sum(rounds[-1]), 4, 128)
    compare(*run(c, torch.from_numpy(q).cuda()), m.attention(q))
    c.close()


@pytest.mark.parametrize("scale", [1e-3, 0.3, 2.0])
def test_scales_and_uneven_pages(tq, scale):
    """Softmaxes from flat to one-hot, and pages whose powers of two differ by far: the largest come first, last and between."""
    rng = np.random.default_rng(11)
    c, m, _ = filled(tq, rng, 2, 128, 16, [[150, 90], [3, 30]], spread=3.0)
    q = queries(rng, 33, 6, 128)
    compare(*run(c, torch.from_numpy(q).cuda(), scale=scale), m.attention(q, scale=float(np.float32(scale))))
    c.close()


@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 20, 90]])
def test_strides_padding_and_rows_left_alone(tq, counts):
    rng = np.random.default_rng(2)
    heads, group, dim = 2, 3, 128
    c, m, rows = filled(tq, rng, heads, dim, 32, [[50, 0, 200]], later=[counts])
    pad = 4
    tokens = sum(counts) + pad
    c.plan(np.array(counts, np.int32), tokens, rows=ints(rows), max_count=200)
    m.plan(counts, rows)
    width = heads * group * dim
    for offset, gap in ((0, 64), (1, 3), (4, 4)):
        flat = torch.tensor(rng.standard_normal((tokens, width + offset + gap)), device="cuda").half()
        flat[-pad:] = float("nan")
        q = flat[:, offset:offset + width].unflatten(1, (heads * group, dim))
        result = torch.full((tokens, width + offset + gap), 9.0, dtype=torch.float16, device="cuda")
        out = result[:, offset:offset + width].unflatten(1, (heads * group, dim))
        lse = torch.full((tokens, heads * group), 9.0, device="cuda")
        c.attention(0, q, out=out, lse=lse)
        compare(out[:-pad], lse[:-pad], m.attention(q[:-pad].cpu().numpy()))
        assert (out[-pad:] == 9).all() and (lse[-pad:] == 9).all() and (result[:, :offset] == 9).all() and (result[:, offset + width:] == 9).all()
    torch.cuda.synchronize()
    c.check_status()
    c.close()


@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("last", [[1, 1], [40, 150]])
def test_pages_that_are_not_numbers(tq, window, dim, last):
    """Rows that see such a page are NaN; those before it, or behind it by more than the window, are not."""
    rng = np.random.default_rng(8)
    c, m, rows = filled(tq, rng, 2, dim, 16, [[30, 77]], later=[[5, 1], last])
    for step, counts in enumerate(([5, 1], last)):
        m.plan(counts, rows)
        c.plan(np.array(counts, np.int32), rows=ints(rows))
        x = [rng.standard_normal((sum(counts), 2, dim)).astype(np.float16) for _ in range(2)]
        if step == 0 or sum(last) > 2:
            x[0][1, 0, 3], x[1][-1, 1, 7] = np.inf, np.nan
        for which in (0, 1):
            m.append(which, x[which])
        c.append(0, torch.from_numpy(x[0]).cuda(), torch.from_numpy(x[1]).cuda())
    q = queries(rng, sum(last), 8, dim)
    want = m.attention(q, window)
    assert np.isnan(want[0]).any() and np.isfinite(want[0]).any()
    compare(*run(c, torch.from_numpy(q).cuda(), window=window), want)
    c.close()


def test_memory_of_earlier_owners_is_not_seen(tq):
    """Pages that held NaNs and large values go to others; their tails are behind the new lengths."""
    rng = np.random.default_rng(4)
    c = tq.PagedKVCache(1, 1, 128, 6, 64, 3, 2, 400)
    m = Model(1, 128, 6, 64)
    c.plan(np.array([128, 128, 128], np.int32))
    m.plan([128] * 3)
    bad = torch.full((384, 1, 128), float("nan"), dtype=torch.float16, device="cuda")
    c.append(0, bad, bad)
    c.truncate(np.zeros(3, np.int32))
    m.truncate([0] * 3)
    for counts in ([70, 1, 10], [1, 1, 1]):
        m.plan(counts)
        c.plan(np.array(counts, np.int32))
        x = [rng.standard_normal((sum(counts), 1, 128)).astype(np.float16) for _ in range(2)]
        m.append(0, x[0])
        m.append(1, x[1])
        c.append(0, torch.from_numpy(x[0]).cuda(), torch.from_numpy(x[1]).cuda())
        q = queries(rng, sum(counts), 5, 128)
        compare(*run(c, torch.from_numpy(q).cuda()), m.attention(q))
    c.close()


def test_results_repeat_to_the_bit(tq):
    rng = np.random.default_rng(6)
    c, _, _ = filled(tq, rng, 2, 128, 64, [[5000, 100, 1300], [1, 30, 200]])
    q = torch.from_numpy(queries(rng, 231, 8, 128)).cuda()
    first = run(c, q)
    for _ in range(5):
        again = run(c, q)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    c.close()


@pytest.mark.parametrize("last", [1, 9])
@pytest.mark.parametrize("big", [2.0 ** 36, 2.0 ** 100])
def test_values_of_any_size(tq, last, big):
    """Most values are zeros, whose pages have the smallest scale there is, one is 2^130 or more above it: sums of weights are what they are without it."""
    rng = np.random.default_rng(12)
    dim, group, tokens = 64, 8, 40000     # (several tiles to a CTA)
    c = tq.PagedKVCache(1, 1, dim, 640, 64, 1, 640, tokens)
    m = Model(1, dim, 640, 64)
    for count in (tokens, last):
        k, v = rng.standard_normal((count, 1, dim)), np.zeros((count, 1, dim))
        if count == tokens:
            k[0, 0] = -4
            v[0, 0] = big
        k, v = k.astype(np.float32), v.astype(np.float32)
        m.plan([count])
        m.append(0, k)
        m.append(1, v)
        c.plan(np.array([count], np.int32))
        c.append(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    q = (2 + 0.1 * rng.standard_normal((last, group, dim))).astype(np.float16)
    out, lse = run(c, torch.from_numpy(q).cuda())
    _, sums, _, ltol = m.attention(q)
    assert (np.abs(lse.cpu().numpy() - sums) <= ltol).all() and not torch.isnan(out).any()
    c.close()


def test_scales_that_vanish(tq):
    """Zero keys and a scale so small that their product is no number of 32 bits: equal weights, and masked tokens are out."""
    c = tq.PagedKVCache(1, 1, 64, 4, 64, 1, 4, 200)
    v = torch.arange(150, device="cuda").half()[:, None, None].expand(150, 1, 64).contiguous()
    c.plan(np.array([150], np.int32))
    c.append(0, torch.zeros_like(v), v)
    q = torch.ones((150, 2, 64), dtype=torch.float16, device="cuda")
    out, lse = run(c, q, scale=1e-30)
    seen = torch.arange(150, device="cuda", dtype=torch.float64)
    codes = torch.cat([torch.round(x / s) * s for x, s in ((seen[:64], 0.5), (seen[64:128], 1.0), (seen[128:], 2.0))])
    mean = torch.cumsum(codes, 0) / (seen + 1)
    # equal weights are halves exactly, sums of codes in halves below 2^16 exact; a division, a product and a half's rounding
    assert (out.double() - mean[:, None, None]).abs().le(mean[:, None, None] * (2.0 ** -11 + 2.0 ** -22)).all()
    # the logarithm of 2^7 n is below 16: a unit of 2^-20 off; the difference and the product with log 2 half a unit below 8 each, 2^-22
    assert (lse.double() - torch.log(seen + 1)[:, None]).abs().le(2.0 ** -19).all()
    c.close()


@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("large", [1e15, 3e38, -3e38])
def test_large_numbers_that_are_not_seen(tq, window, large):
    """Tokens from the 129th on are as large as they can be: the rows before them, in the same tile, are what they are without."""
    rng = np.random.default_rng(13)
    c = tq.PagedKVCache(1, 1, 128, 8, 64, 1, 8, 250)
    m = Model(1, 128, 8, 64)
    k, v = rng.standard_normal((250, 1, 128)).astype(np.float32), rng.standard_normal((250, 1, 128)).astype(np.float32)
    k[128:] = v[128:] = large
    m.plan([250])
    c.plan(np.array([250], np.int32))
    c.append(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    q = queries(rng, 250, 1, 128)
    out, lse = run(c, torch.from_numpy(q).cuda(), window=window)
    m = Model(1, 128, 8, 64)
    m.plan([128])
    m.append(0, k[:128])
    m.append(1, v[:128])
    compare(out[:128], lse[:128], m.attention(q[:128], window))
    c.close()
