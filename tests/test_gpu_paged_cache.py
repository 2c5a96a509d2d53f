"""GPU tests of the paged cache's plans, truncations, appends and page reads: equal to the definitions, bit for bit."""
import numpy as np
import pytest

from tests.paged_model import Model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


class Outputs:
    def __init__(self, n, tokens, width):
        self.arrays = {"starts": torch.full((n + 1,), 77, dtype=torch.int32, device="cuda"), "lengths": torch.full((n,), 77, dtype=torch.int32, device="cuda"),
                       "slots": torch.full((tokens,), 77, dtype=torch.int32, device="cuda"),
                       "positions": torch.full((tokens,), 77, dtype=torch.int32, device="cuda"),
                       "tables": torch.full((n, width), 77, dtype=torch.int32, device="cuda")}

    def check(self, model, rows, counts, slots, positions):
        got = {k: v.cpu().numpy() for k, v in self.arrays.items()}
        assert got["starts"].tolist() == [0, *np.cumsum(counts)]
        assert got["lengths"].tolist() == [model.lengths[r] for r in rows]
        pad = len(got["slots"]) - len(slots)
        assert got["slots"].tolist() == slots + [-1] * pad and got["positions"].tolist() == positions + [0] * pad
        width = got["tables"].shape[1]
        assert got["tables"].tolist() == [(model.tables[r] + [-1] * width)[:width] for r in rows]


@pytest.mark.parametrize("page,requests,most,steps,pad,width", [
    (16, 1, 1, 40, 0, 4), (16, 7, 40, 12, 3, 30), (64, 33, 200, 6, 1, 2), (128, 300, 3, 8, 0, 9), (32, 1025, 7, 5, 5, 3), (16, 4096, 2, 3, 0, 1), (64, 5, 30000, 2, 0, 1000)])
def test_plans_and_truncations(tq, page, requests, most, steps, pad, width):
    rng = np.random.default_rng(page + requests)
    room = steps * most // page + 1
    pages = requests * room if requests * room < 60000 else 60000
    c = tq.PagedKVCache(1, 1, 64, pages, page, requests, room, requests * most + pad)
    m = Model(1, 64, 1, page)
    m.stack = list(range(pages))[::-1]
    for step in range(steps):
        n = requests if step % 2 == 0 else max(1, requests // 2)
        rows = rng.permutation(requests)[:n].tolist()
        counts = rng.integers(0, most + 1, n)
        total = int(counts.sum()) + pad
        out = Outputs(n, total, width)
        slots, positions = m.plan(counts.tolist(), rows)
        c.plan(ints(counts) if step % 3 else counts.astype(np.int32), total, most, rows=ints(rows), **out.arrays)
        out.check(m, rows, counts, slots, positions)
        if step % 2:
            keep = [int(rng.integers(0, m.lengths[r] + 1)) if rng.random() < 0.5 else m.lengths[r] for r in rows]
            m.truncate(keep, rows)
            c.truncate(ints(keep) if step % 3 else np.array(keep, np.int32), rows=ints(rows))
    torch.cuda.synchronize()
    c.check_status()
    assert c.free_pages() == len(m.stack)
    c.close()


def test_plan_without_rows_or_requests(tq):
    c = tq.PagedKVCache(1, 1, 64, 8, 16, 4, 4, 64)
    out = Outputs(3, 9, 4)
    c.plan(np.array([4, 0, 5], np.int32), **out.arrays)
    m = Model(1, 64, 8, 16)
    out.check(m, [0, 1, 2], [4, 0, 5], *m.plan([4, 0, 5]))
    empty = Outputs(0, 6, 4)
    c.plan(np.zeros(0, np.int32), 6, **{k: v for k, v in empty.arrays.items() if k in ("starts", "slots", "positions")})
    assert empty.arrays["starts"].tolist() == [0] and empty.arrays["slots"].tolist() == [-1] * 6 and empty.arrays["positions"].tolist() == [0] * 6
    zeros = torch.zeros((6, 1, 64), dtype=torch.float16, device="cuda")
    c.append(0, zeros, zeros)
    c.attention(0, zeros)
    c.truncate(np.zeros(0, np.int32))
    torch.cuda.synchronize()
    c.check_status()
    assert c.free_pages() == 6
    c.close()


@pytest.mark.parametrize("rows,counts,tokens,most,what", [
    ([0, 4], [1, 1], 9, 9, "row"), ([-1, 2], [1, 1], 9, 9, "row"), ([2, 2], [1, 1], 9, 9, "row"), ([0, 1], [1, -1], 9, 9, "count"),
    ([0, 1], [1, 6], 9, 5, "count"), ([0, 1], [5, 5], 9, 5, "count"), ([0, 1], [46, 1], 99, 99, "max_pages"), ([1, 0, 2, 3], [33, 9, 48, 48], 199, 99, "free pages"),
    ([0, 1], [2147483647, 2147483647], 199, 2147483647, "max_pages")])
def test_plans_that_do_not_fit(tq, rows, counts, tokens, most, what):
    """Nothing changes, the outputs are those of an empty batch, and the step's calls do nothing."""
    c = tq.PagedKVCache(1, 2, 64, 9, 16, 4, 3, 200)
    m = Model(2, 64, 9, 16)
    rng = np.random.default_rng(0)
    x = torch.tensor(rng.standard_normal((20, 2, 64)), device="cuda").half()
    m.plan([5, 15])
    c.plan(np.array([5, 15], np.int32))
    c.append(0, x, x)
    m.append(0, x.cpu().numpy())
    out = Outputs(len(rows), tokens, 3)
    c.plan(ints(counts), tokens, most, rows=ints(rows), **out.arrays)
    big = torch.full((tokens, 2, 64), 3.0, dtype=torch.float16, device="cuda")
    c.append(0, big, big)
    result = c.attention(0, big, out=torch.full_like(big, 7.0))
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match=what):
        c.check_status()
    torch.cuda.synchronize()
    c.check_status()
    assert out.arrays["starts"].tolist() == [0] * (len(rows) + 1)
    assert (out.arrays["slots"] == -1).all() and (out.arrays["positions"] == 0).all() and (result == 7).all()
    assert c.free_pages() == 7
    pages = ints(range(9))
    k = torch.empty((9, 16, 2, 64), device="cuda")
    c.read_pages(0, pages, k)
    assert np.array_equal(k.cpu().numpy(), m.values(0, range(9)))
    # truncations
    for keep, named in (([6], [0]), ([-1], [0]), ([1, 1], [0, 0]), ([1], [7])):
        c.truncate(ints(keep), rows=ints(named))
        torch.cuda.synchronize()
        with pytest.raises(tq.TQError):
            c.check_status()
    assert c.free_pages() == 7
    slots, positions = m.plan([20, 1])
    out = Outputs(2, 21, 3)
    c.plan(np.array([20, 1], np.int32), **out.arrays)
    out.check(m, [0, 1], [20, 1], slots, positions)
    torch.cuda.synchronize()
    c.check_status()
    c.close()


def refused_calls(c, x):
    """(error, what it says, call), on a cache of one layer of 2 heads of 64 dims with a plan of 3 tokens."""
    wide = torch.zeros((3, 2, 128), dtype=torch.float16, device="cuda")
    host = np.zeros((3, 2, 64), np.float16)
    return [
        (ValueError, "tokens", lambda: c.plan(ints([1]))), (TypeError, "int32", lambda: c.plan(torch.zeros(1, dtype=torch.long, device="cuda"), 1, 1)),
        (ValueError, "slots", lambda: c.plan(np.ones(1, np.int32), slots=ints([1, 2]))), (ValueError, "width", lambda: c.plan(np.ones(1, np.int32), tables=ints([[1], [2]]))),
        (Exception, "more requests", lambda: c.plan(np.ones(5, np.int32))), (Exception, "more tokens", lambda: c.plan(np.array([201], np.int32))),
        (Exception, "negative", lambda: c.plan(np.ones(1, np.int32), 1, -1)), (Exception, "device pointers", lambda: c.plan(np.ones(1, np.int32), slots=np.zeros(1, np.int32))),
        (ValueError, "must be", lambda: c.append(0, x[:, :1], x[:, :1])), (ValueError, "same number", lambda: c.append(0, x, x[:2])), (ValueError, "same number", lambda: c.append(0, x, x.float())),
        (TypeError, "float", lambda: c.append(0, x.bfloat16(), x.bfloat16())), (TypeError, "torch", lambda: c.append(0, host, host)), (Exception, "Layer", lambda: c.append(1, x, x)),
        (Exception, "Layer", lambda: c.append(-1, x, x)), (Exception, "plan is for 3", lambda: c.append(0, x[:2], x[:2])),
        (Exception, "device pointers", lambda: c.append(0, x.cpu(), x.cpu())), (ValueError, "contiguous", lambda: c.append(0, wide[:, :, ::2], x)),
        (TypeError, "float16", lambda: c.attention(0, x.float())), (ValueError, "must be", lambda: c.attention(0, wide)), (Exception, "multiple", lambda: c.attention(0, x[:, :1])),
        (Exception, "window", lambda: c.attention(0, x, window=-1)), (Exception, "scale", lambda: c.attention(0, x, scale=float("nan"))),
        (Exception, "scale", lambda: c.attention(0, x, scale=-1.0)), (ValueError, "lse", lambda: c.attention(0, x, lse=torch.zeros(3, device="cuda"))),
        (ValueError, "out", lambda: c.attention(0, x, out=torch.zeros_like(x[:2]))), (Exception, "Layer", lambda: c.attention(2, x)),
        (Exception, "plan is for 3", lambda: c.attention(0, x[:2])), (Exception, "device pointers", lambda: c.attention(0, x.cpu())),
        (ValueError, "contiguous", lambda: c.read_pages(0, ints([0]), x)), (ValueError, "same type", lambda: c.read_pages(
            0, ints([0]), torch.zeros((1, 16, 2, 64), device="cuda"), torch.zeros((1, 16, 2, 64), device="cuda").half())),
    ]


def test_calls_that_are_refused(tq):
    c = tq.PagedKVCache(1, 2, 64, 9, 16, 4, 3, 200)
    x = torch.ones((3, 2, 64), dtype=torch.float16, device="cuda")
    for call in (lambda: c.append(0, x, x), lambda: c.attention(0, x)):
        with pytest.raises(tq.TQError, match="no plan"):
            call()
    c.plan(np.array([3], np.int32))
    for kind, what, call in refused_calls(c, x):
        with pytest.raises(kind, match=what):
            call()
    c.append(0, x, x)
    out = c.attention(0, x)
    assert torch.equal(out, x)       # equal values: whatever the weights
    # a page number outside the cache leaves its rows as they are
    k = torch.full((3, 16, 2, 64), 5.0, device="cuda")
    c.read_pages(0, ints([0, 9, -1]), k)
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="page number"):
        c.check_status()
    assert (k[0, :3] == 1).all() and (k[0, 3:] == 0).all() and (k[1:] == 5).all()
    c.truncate(np.zeros(1, np.int32))
    with pytest.raises(tq.TQError, match="no plan"):
        c.append(0, x, x)
    c.close()


def rows_of(rng, kind, tokens, heads, dim, dtype):
    """Keys or values whose scales grow, shrink and meet the borders."""
    x = rng.standard_normal((tokens, heads, dim)) * np.exp2(rng.integers(-6, 7, (tokens, heads, 1)))
    if kind == "borders":     # magnitudes at which the power of two changes, and halves that go to the even number
        x = rng.integers(-255, 256, x.shape) / 2.0 * np.exp2(rng.integers(-3, 4, (tokens, 1, 1)))
    elif kind == "small":     # subnormal halves, zero rows; in fp32 numbers below the smallest scale
        x = x * 2.0 ** (-22 if dtype == np.float16 else -104)
        x[rng.random(tokens) < 0.3] = 0
    elif kind == "large":
        x = np.clip(x * (2000 if dtype == np.float16 else 2.0 ** 118), -65504 if dtype == np.float16 else -3.4e38, 65504 if dtype == np.float16 else 3.4e38)
    return x.astype(dtype)


@pytest.mark.parametrize("dim,page", [(64, 16), (64, 128), (128, 32), (128, 64)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("kind", ["plain", "borders", "small", "large"])
def test_appends_hold_the_defined_codes(tq, dim, page, dtype, kind):
    """Chunks, single tokens and drafts that are taken back, in pages that requests take and leave."""
    rng = np.random.default_rng(dim + page)
    heads, requests = 3, 4
    pages = requests * (600 // page + 2)
    c = tq.PagedKVCache(2, heads, dim, pages, page, requests, 600 // page + 2, 1000)
    m = Model(heads, dim, pages, page)
    for step, counts in enumerate([[70, 1, 0, 17], [1, 1, 1, 1], [9, 130, 2, 0], [1, 0, 1, 1], [3, 3, 5, 8], [140, 1, 33, 64], [1, 1, 1, 1]]):
        rows = rng.permutation(requests).tolist()
        m.plan(counts, rows)
        c.plan(np.array(counts, np.int32), rows=ints(rows))
        k, v = (rows_of(rng, kind, sum(counts), heads, dim, dtype) for _ in range(2))
        c.append(1, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
        m.append(0, k)
        m.append(1, v)
        if step in (2, 4):
            keep = [max(0, m.lengths[r] - 5) if r % 2 else m.lengths[r] for r in range(requests)]
            m.truncate(keep)
            c.truncate(np.array(keep, np.int32))
        out = [torch.empty((pages, page, heads, dim), device="cuda") for _ in range(2)]
        c.read_pages(1, ints(range(pages)), *out)
        for which in (0, 1):
            assert np.array_equal(out[which].cpu().numpy().astype(np.float64), m.values(which, range(pages))), (step, which)
    half = [torch.empty((2, page, heads, dim), dtype=torch.float16, device="cuda") for _ in range(2)]
    mine = [m.tables[0][-1], m.tables[3][0]]
    c.read_pages(1, ints(mine), *half)
    for which in (0, 1):
        with np.errstate(over="ignore"):
            assert np.array_equal(half[which].cpu().numpy(), m.values(which, mine).astype(np.float16))
    other = torch.empty((pages, page, heads, dim), device="cuda")
    c.read_pages(0, ints(range(pages)), None, other)
    assert (other == 0).all()
    torch.cuda.synchronize()
    c.check_status()
    c.close()


@pytest.mark.parametrize("counts", [[5, 1, 40], [1, 1, 1]])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("offset,gap", [(0, 0), (0, 8), (1, 0), (3, 5), (8, 16)])
def test_appends_of_strided_rows(tq, counts, dtype, offset, gap):
    """Slices of a fused projection's rows, aligned or not, with rows behind the last request's."""
    rng = np.random.default_rng(offset + gap)
    heads, dim, page = 2, 128, 16
    tokens = sum(counts) + 2
    c = tq.PagedKVCache(1, heads, dim, 8, page, 3, 4, 100)
    m = Model(heads, dim, 8, page)
    width = heads * dim
    flat = torch.tensor(rng.standard_normal((tokens, 2 * width + gap + offset)), device="cuda").to(dtype)
    flat[-2:] = float("nan")
    k = flat[:, offset:offset + width].unflatten(1, (heads, dim))
    v = flat[:, offset + width:offset + 2 * width].unflatten(1, (heads, dim))
    c.plan(np.array(counts, np.int32), tokens)
    m.plan(counts)
    c.append(0, k, v)
    out = [torch.empty((8, page, heads, dim), device="cuda") for _ in range(2)]
    c.read_pages(0, ints(range(8)), *out)
    for which, x in enumerate((k, v)):
        m.append(which, x[:-2].cpu().numpy())
        assert np.array_equal(out[which].cpu().numpy().astype(np.float64), m.values(which, range(8)))
    torch.cuda.synchronize()
    c.check_status()
    c.close()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("many", [False, True])
def test_values_that_are_not_finite_mark_their_page_and_head(tq, dtype, many):
    heads, dim, page = 3, 64, 16
    c = tq.PagedKVCache(1, heads, dim, 6, page, 2, 3, 64)
    m = Model(heads, dim, 6, page)
    rng = np.random.default_rng(3)
    for counts in ([20, 9] if many else [2, 1], [1, 1], [20, 3] if many else [1, 2]):
        x = torch.tensor(rng.standard_normal((sum(counts), heads, dim)), device="cuda").to(dtype)
        y = x * 2
        if counts == [1, 1]:
            x[0, 1, 5], y[1, 2, 63] = float("nan"), float("-inf")
        c.plan(np.array(counts, np.int32))
        m.plan(counts)
        c.append(0, x, y)
        m.append(0, x.cpu().numpy())
        m.append(1, y.cpu().numpy())
    out = [torch.empty((6, page, heads, dim), device="cuda") for _ in range(2)]
    c.read_pages(0, ints(range(6)), *out)
    for which in (0, 1):
        want = m.values(which, range(6))
        assert np.isnan(want).any() and np.array_equal(out[which].cpu().numpy().astype(np.float64), want, equal_nan=True)
    # the pages are begun anew
    c.truncate(np.zeros(2, np.int32))
    m.truncate([0, 0])
    x = torch.ones((48, heads, dim), dtype=dtype, device="cuda")
    c.plan(np.array([24, 24], np.int32))
    m.plan([24, 24])
    c.append(0, x, x)
    c.read_pages(0, ints(m.tables[0] + m.tables[1]), *(o[:4] for o in out))
    assert torch.isfinite(out[0][:4]).all() and torch.isfinite(out[1][:4]).all()
    c.close()
