"""GPU tests of attention of trees of drafts over the paged cache against its definition in 64 bits, within bounds that follow from the roundings."""
import numpy as np
import pytest

from tests import tree_attention_model
from tests.drafts_model import trees
from tests.paged_model import Model
from tests.test_gpu_paged_attention import compare, ints, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class Batch:
    """A cache of one layer and its model: what requests hold, and trees of drafts behind it."""

    def __init__(self, tq, rng, heads, dim, page, held, counts, spread, pad=0, strength=1.0, key=None, value=None):
        n, pages = len(held), sum(-(-(h + c) // page) for h, c in zip(held, counts)) + 3
        self.c = tq.PagedKVCache(1, heads, dim, pages, page, n, pages, max(sum(held), sum(counts)) + pad + 8)
        self.m = Model(heads, dim, pages, page)
        rows = rng.permutation(n).tolist()
        self.parents = trees(rng, counts, spread)
        for new in (held, counts):
            last = new is counts
            self.m.plan(new, rows)
            self.c.plan(np.array(new, np.int32), sum(new) + (pad if last else 0), rows=ints(rows))
            kv = []
            for which, change in ((0, key), (1, value)):
                x = rng.standard_normal((sum(new), heads, dim)) * np.exp(strength * rng.standard_normal((sum(new), 1, 1)))
                if change is not None:
                    x = change(x, last)
                kv.append(x.astype(np.float32))
                self.m.append(which, kv[-1])
            if last:
                flat = np.concatenate([np.asarray(p, np.int32) for p in self.parents] + [np.full(pad, -7, np.int32)])
                self.positions = torch.zeros(sum(new) + pad, dtype=torch.int32, device="cuda")
                self.c.tree(ints(flat), positions=self.positions)
                kv = [np.concatenate([x, np.zeros((pad, heads, dim), np.float32)]) for x in kv]
            if sum(new):
                self.c.append(0, *(torch.from_numpy(x).cuda() for x in kv))
        self.tokens, self.pad = sum(counts), pad

    def run(self, q, **more):
        lse = torch.full(q.shape[:2], 9.0, device="cuda")
        out = self.c.tree_attention(0, q, out=torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda"), lse=lse, **more)
        torch.cuda.synchronize()
        self.c.check_status()
        return out, lse

    def check(self, rng, group, window=0, scale=0.0, q=None):
        heads, dim = self.m.heads, self.m.dim
        q = queries(rng, self.tokens + self.pad, heads * group, dim) if q is None else q
        out, lse = self.run(torch.from_numpy(q).cuda(), window=window, scale=scale)
        if self.pad:
            assert (out[self.tokens:] == 9).all() and (lse[self.tokens:] == 9).all()
        compare(out[:self.tokens], lse[:self.tokens], tree_attention_model.attention(self.m, q[:self.tokens], self.parents, window, scale or None))
        return out, lse


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("page", [64, 16, 32, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 7), (3, 5), (1, 16), (2, 24)])
def test_trees(tq, dim, page, heads, group):
    rng = np.random.default_rng(dim + page + group)
    b = Batch(tq, rng, heads, dim, page, [0, 1, 15, 16, 127, 128, 200, 333, 0], [1, 5, 16, 3, 9, 1, 8, 12, 0], 3)
    b.check(rng, group)
    b.c.close()


@pytest.mark.parametrize("dim,page,heads,group", [(128, 64, 2, 7), (64, 32, 2, 4), (128, 16, 1, 8), (64, 64, 1, 40)])
@pytest.mark.parametrize("held,counts,spread", [
    ([0], [1], 1), ([0], [200], 5), ([130], [64], 4), ([1000], [31], 300), ([77] * 20, [3] * 20, 2), ([255, 256, 257], [1, 1, 1], 1), ([5, 700], [256, 2], 40),
    ([120], [300], 0), ([3000], [2], 2)])
def test_shapes_of_batches(tq, dim, page, heads, group, held, counts, spread):
    rng = np.random.default_rng(dim + group)
    b = Batch(tq, rng, heads, dim, page, held, counts, spread, pad=2)
    b.check(rng, group)
    b.c.close()


@pytest.mark.parametrize("window", [1, 2, 7, 64, 128, 129, 300, 100000])
@pytest.mark.parametrize("dim,page,group", [(128, 64, 4), (64, 16, 7)])
def test_windows(tq, window, dim, page, group):
    rng = np.random.default_rng(window)
    b = Batch(tq, rng, 2, dim, page, [0, 5, 130, 127, 600], [9, 17, 30, 4, 40], 4)
    b.check(rng, group, window=window)
    b.c.close()


def test_chains_are_causal(tq):
    """The same definition, and the causal kernels' results: each of the two is within its own bound of it, so that they are within both
    together of each other (a bound that does not go by the numbers' size, 0.02, is less than half a step of a half of 43)."""
    rng = np.random.default_rng(1)
    b = Batch(tq, rng, 2, 128, 64, [100, 0, 500], [9, 17, 1], 1)
    q = queries(rng, 27, 8, 128)
    out, lse = b.check(rng, 4, q=q)
    want, sums, tol, ltol = b.m.attention(q)
    mine = tree_attention_model.attention(b.m, q, b.parents)
    assert np.abs(mine[0] - want).max() < 1e-9 and np.abs(mine[1] - sums).max() < 1e-9
    log = torch.zeros((27, 8), device="cuda")
    causal = b.c.attention(0, torch.from_numpy(q).cuda(), lse=log)
    assert (np.abs((causal.float() - out.float()).cpu().numpy()) <= tol + mine[2]).all() and (np.abs((log - lse).cpu().numpy()) <= ltol + mine[3]).all()
    b.c.close()


def test_long_contexts_in_parts(tq):
    """Few items over many tiles: each is cut into many parts; the same again, bit for bit."""
    rng = np.random.default_rng(2)
    b = Batch(tq, rng, 1, 64, 128, [40000, 17000], [8, 3], 3)
    q = queries(rng, 11, 4, 64)
    first = b.check(rng, 4, q=q)
    again = b.run(torch.from_numpy(q).cuda())
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    b.c.close()


@pytest.mark.parametrize("scale", [1e-6, 0.3, 3.0, 40.0])
def test_scales_and_references_that_move(tq, scale):
    """Keys that grow along the context: every tile has larger scores than all before, up to thousands of powers of two."""
    rng = np.random.default_rng(3)
    grow = lambda x, last: x * (np.linspace(0.2, 4, len(x))[:, None, None] if not last else 4)      # noqa: E731
    b = Batch(tq, rng, 2, 64, 32, [1500], [12], 3, strength=0.1, key=grow)
    b.check(rng, 5, scale=scale)
    b.c.close()


@pytest.mark.parametrize("low,high", [(-2, 2), (-30, 10), (-75, 3), (-20, 100)])
def test_values_far_apart(tq, low, high):
    """Values whose scales lie up to 2^120 apart from page to page."""
    rng = np.random.default_rng(high)

    def apart(x, last):
        e = np.repeat(rng.integers(low, high + 1, len(x) // 16 + 1), 16)[:len(x)]
        return np.ldexp(x, e[:, None, None])
    b = Batch(tq, rng, 1, 64, 16, [600, 16], [20, 20], 4, strength=0.0, value=apart)
    q = queries(rng, 40, 3, 64)
    out, lse = b.run(torch.from_numpy(q).cuda())
    want, sums, tol, ltol = tree_attention_model.attention(b.m, q, b.parents)
    got = out.cpu().numpy().astype(np.float64)
    beyond = np.abs(want) + tol > 65504       # (more than a half holds)
    assert np.isfinite(got[~beyond]).all() and (np.abs(got - want) <= tol)[~beyond].all()
    assert (np.abs(lse.cpu().numpy() - sums) <= ltol).all()
    b.c.close()


def test_large_numbers_that_a_row_does_not_see(tq):
    """A draft with keys and values 2^60 above all others in a page of its own: those beside it are as if it were not there."""
    rng = np.random.default_rng(5)
    held, counts = [64], [48]

    def large(x, last):
        if last:
            x[16:32] *= 2.0 ** 60      # nodes 16 .. 31: a page
        return x
    b = Batch(tq, rng, 1, 64, 16, held, counts, 1, strength=0.2, value=large)
    b.parents[0] = [-1] + [j - 1 if j % 16 else 0 for j in range(1, 48)]       # three branches
    b.c.tree(ints(b.parents[0]))
    q = queries(rng, 48, 4, 64)
    out, lse = b.run(torch.from_numpy(q).cuda())
    want, sums, tol, ltol = tree_attention_model.attention(b.m, q, b.parents)
    away = [j for j in range(48) if not 16 <= j < 32]
    assert (np.abs(out.cpu().numpy() - want) <= tol)[away].all() and (np.abs(lse.cpu().numpy() - sums) <= ltol).all()
    b.c.close()


def test_pages_that_are_not_numbers(tq):
    """Rows that see a token of such a page and head are not numbers, the others are as they were."""
    rng = np.random.default_rng(6)

    def bad(x, last):
        if last:
            x[17, 0, 3], x[33, 1, 0] = np.nan, np.inf
        return x
    for which in ("key", "value"):
        b = Batch(tq, rng, 2, 64, 16, [48], [48], 1, **{which: bad})
        b.parents[0] = [-1] + [j - 1 if j % 16 else 0 for j in range(1, 48)]
        b.c.tree(ints(b.parents[0]))
        out, _ = b.check(rng, 3)
        lost = torch.isnan(out).any(2)
        assert lost[16:32, :3].all() and not lost[16:32, 3:].any() and lost[32:, 3:].all() and not lost[:16].any()
        b.c.close()
    # and an older one, which all see
    b = Batch(tq, rng, 2, 64, 16, [48], [4], 1, value=lambda x, last: x if last else np.where(np.arange(48)[:, None, None] == 20, np.nan, x))
    assert torch.isnan(b.check(rng, 3)[0]).all()
    b.c.close()


def test_queries_that_are_not_numbers(tq):
    rng = np.random.default_rng(7)
    b = Batch(tq, rng, 1, 128, 64, [300], [9], 2)
    q = queries(rng, 9, 4, 128)
    want = b.check(rng, 4, q=q)[0]
    q[2, 1, 5], q[4, 0, 0] = np.nan, np.inf
    out, lse = b.run(torch.from_numpy(q).cuda())
    lost = torch.isnan(out).any(2)
    assert lost[2, 1] and lost[4, 0] and int(lost.sum()) == 2 and torch.isnan(lse[2, 1]) and torch.equal(out[~lost], want[~lost])
    b.c.close()


@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 0), (4, 8), (8, 24)])
def test_strides_and_alignment(tq, shift, pad):
    rng = np.random.default_rng(8)
    b = Batch(tq, rng, 2, 64, 32, [77, 200], [9, 20], 3)
    q = queries(rng, 29, 6, 64)
    want = b.check(rng, 3, q=q)
    room = [torch.full((shift + 29 * (6 * 64 + pad) + 16,), 5.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    view = [x[shift:].as_strided((29, 6, 64), (6 * 64 + pad, 64, 1)) for x in room]
    view[0].copy_(torch.from_numpy(q))
    lse = torch.zeros((29, 6), device="cuda")
    b.c.tree_attention(0, view[0], out=view[1], lse=lse)
    assert torch.equal(view[1], want[0]) and torch.equal(lse, want[1])
    rest = torch.cat([room[1][:shift], room[1][shift:].as_strided((29, pad), (6 * 64 + pad, 1), shift + 6 * 64).flatten()])
    assert (rest == 5).all()
    b.c.close()


def test_requests_whose_parents_are_no_tree_are_left_alone(tq):
    rng = np.random.default_rng(9)
    b = Batch(tq, rng, 1, 64, 16, [20, 30, 40], [4, 5, 6], 2)
    q = torch.from_numpy(queries(rng, 15, 2, 64)).cuda()
    want, _ = b.run(q)
    bad = [x for p in b.parents for x in p]
    bad[7] = 4
    b.c.tree(ints(bad))
    out = b.c.tree_attention(0, q, out=torch.full_like(q, 3.0))
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="tree"):
        b.c.check_status()
    assert torch.equal(out[:4], want[:4]) and (out[4:9] == 3).all() and torch.equal(out[9:], want[9:])
    b.c.close()


def test_calls_out_of_turn(tq):
    c = tq.PagedKVCache(1, 2, 64, 8, 16, 2)
    q = torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(tq.TQError, match="no plan"):
        c.tree_attention(0, q)
    c.plan([3])
    with pytest.raises(tq.TQError, match="no trees"):
        c.tree_attention(0, q)
    c.tree()
    c.append(0, q, q)
    c.tree_attention(0, q)
    c.attention(0, q)           # (a plan with trees has both)
    c.plan([3])
    with pytest.raises(tq.TQError, match="no trees"):
        c.tree_attention(0, q)
    for bad in (lambda: c.tree_attention(0, q.float()), lambda: c.tree_attention(0, q[:, :, :32]), lambda: c.tree_attention(0, q, lse=torch.zeros((3, 3), device="cuda"))):
        with pytest.raises((TypeError, ValueError)):
            bad()
    torch.cuda.synchronize()
    c.check_status()
    c.close()


def test_a_replayed_plan_without_trees(tq):
    """Behind a replayed plan of the same sizes that has no trees a call does nothing, and the status tells."""
    rng = np.random.default_rng(10)
    c = tq.PagedKVCache(1, 1, 64, 40, 16, 2)
    q = torch.from_numpy(queries(rng, 6, 2, 64)).cuda()
    k = q[:, :1].contiguous()
    counts = ints([3, 3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.plan(counts, 6, 3, stream=side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.plan(counts, 6, 3, stream=side)
        c.plan(counts, 6, 3, stream=side)
        c.tree(stream=side)
        c.append(0, k, k, stream=side)
        graph.replay()
        out = c.tree_attention(0, q, out=torch.full_like(q, 3.0), stream=side)
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="plan on the device"):
        c.check_status()
    assert (out == 3).all()
    c.close()


def test_captured_and_replayed_on_new_trees(tq):
    rng = np.random.default_rng(11)
    b = Batch(tq, rng, 2, 128, 32, [150, 60, 7], [12, 9, 3], 3)
    q = torch.from_numpy(queries(rng, 24, 8, 128)).cuda()
    parents, out, lse = ints([x for p in b.parents for x in p]), torch.zeros_like(q), torch.zeros((24, 8), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b.c.tree(parents, stream=side)
            b.c.tree_attention(0, q, out=out, lse=lse, stream=side)
    for spread in (1, 2, 9):
        b.parents = trees(rng, [12, 9, 3], spread)
        parents.copy_(ints([x for p in b.parents for x in p]))
        x = queries(rng, 24, 8, 128)
        q.copy_(torch.from_numpy(x))
        graph.replay()
        torch.cuda.synchronize()
        compare(out, lse, tree_attention_model.attention(b.m, x, b.parents))
    b.c.check_status()
    b.c.close()


def test_two_caches_on_two_streams(tq):
    """Calls of two caches at once, several of each behind one another: each has the result that it has alone."""
    rng = np.random.default_rng(12)
    batches = [Batch(tq, rng, 2, 128, 64, [700, 130, 5], [12, 40, 3], 3), Batch(tq, rng, 4, 64, 16, [90] * 9, [7] * 9, 2)]
    qs = [torch.from_numpy(queries(rng, b.tokens, g, b.m.dim)).cuda() for b, g in zip(batches, (8, 4))]
    alone = [b.run(q) for b, q in zip(batches, qs)]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(20):
        outs = []
        for b, q, stream in zip(batches, qs, streams):
            with torch.cuda.stream(stream):
                out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda")
                for _ in range(3):
                    b.c.tree_attention(0, q, out=out, lse=lse, stream=stream)
                outs.append((out, lse))
        torch.cuda.synchronize()
        for (out, lse), (want, sums) in zip(outs, alone):
            assert torch.equal(out, want) and torch.equal(lse, sums)
    for b in batches:
        b.c.check_status()
        b.c.close()
