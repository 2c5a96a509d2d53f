"""GPU tests of the paged cache as a server uses it: requests that come, grow, take drafts back and go, over several layers, eagerly, on other
streams and as captured steps."""
import numpy as np
import pytest

from tests.paged_model import Model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def within(got, lse, want):
    out, sums, tol, ltol = want
    got, lse = got.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    assert (np.abs(got - out) <= tol).all() and (np.abs(lse - sums) <= ltol).all()


# Requests by row: (rows, counts, lengths that truncation leaves behind the step or None, window)
STEPS = [
    ([0, 2], [70, 3], None, 0),                       # two prompts
    ([0, 2, 1], [1, 1, 150], None, 0),                # decode beside a prompt
    ([1, 0, 2], [40, 1, 1], None, 48),                # ... beside its second chunk, in a window
    ([0, 1, 2], [5, 5, 5], [72, 195, 6], 0),          # drafts, of which some are kept
    ([0, 1, 2], [1, 1, 1], [0, 196, 7], 0),           # the first request goes
    ([3, 2, 1, 0], [33, 1, 1, 2], None, 0),           # others take its pages
    ([0, 1, 2, 3], [4, 4, 4, 4], [6, 199, 11, 36], 7),
    ([0, 1, 2, 3], [1, 0, 1, 1], None, 0),
]


@pytest.mark.parametrize("dim,page,heads,group", [(128, 16, 2, 5), (64, 64, 1, 8), (128, 128, 2, 1)])
def test_a_served_batch(tq, dim, page, heads, group):
    """Rotary embedding by the plan's positions, appends of a fused projection's slices, attention, in two layers with values of their own."""
    L = tq.load()
    rng = np.random.default_rng(dim + page)
    layers, pages = 2, sum(-(-x // page) for x in (80, 210, 20, 60))
    c = tq.PagedKVCache(layers, heads, dim, pages, page, 4, 220 // page + 1, 200)
    models = [Model(heads, dim, pages, page) for _ in range(layers)]
    for rows, counts, keep, window in STEPS:
        tokens, pad = sum(counts), 2
        positions, slots = (torch.full((tokens + pad,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
        c.plan(np.array(counts, np.int32), tokens + pad, max(counts), rows=ints(rows), positions=positions, slots=slots)
        wanted = [m.plan(counts, rows) for m in models][0]
        assert slots.tolist() == wanted[0] + [-1] * pad and positions.tolist() == wanted[1] + [0] * pad
        for layer, m in enumerate(models):
            q_heads = heads * group
            fused = torch.from_numpy(rng.standard_normal((tokens + pad, q_heads + 2 * heads, dim)).astype(np.float16)).cuda()
            q, k, v = fused[:, :q_heads].contiguous(), fused[:, q_heads:q_heads + heads].contiguous(), fused[:, q_heads + heads:]
            assert L.tq_rope_qk_f16(q.data_ptr(), k.data_ptr(), positions.data_ptr(), tokens + pad, q_heads, heads, dim, 10000.0, None) == 0
            c.append(layer, k, v)
            lse = torch.full((tokens + pad, q_heads), 9.0, device="cuda")
            out = c.attention(layer, q, window=window, out=torch.full_like(q, 9.0), lse=lse)
            m.append(0, k[:tokens].cpu().numpy())
            m.append(1, v[:tokens].cpu().numpy())
            within(out[:tokens], lse[:tokens], m.attention(q[:tokens].cpu().numpy(), window))
            assert (out[tokens:] == 9).all() and (lse[tokens:] == 9).all()
        if keep is not None:
            c.truncate(np.array(keep, np.int32), rows=ints(rows))
            for m in models:
                m.truncate(keep, rows)
        torch.cuda.synchronize()
        c.check_status()
        assert c.free_pages() == len(models[0].stack)
    for layer, m in enumerate(models):
        k, v = (torch.empty((pages, page, heads, dim), device="cuda") for _ in range(2))
        c.read_pages(layer, ints(range(pages)), k, v)
        used = [p for t in m.tables.values() for p in t]
        for which, x in enumerate((k, v)):
            assert np.array_equal(x.cpu().numpy()[used].astype(np.float64), m.values(which, used))
    c.close()


class Step:
    """Buffers of a step of n requests of up to `most` tokens: a server's, the same in every replay."""

    def __init__(self, n, most, heads, group, dim, layers):
        t = n * most
        self.n, self.most, self.tokens = n, most, t
        self.counts, self.keep, self.rows = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
        self.starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.slots, self.positions = (torch.zeros(t, dtype=torch.int32, device="cuda") for _ in range(2))
        self.tables = torch.zeros((n, 12), dtype=torch.int32, device="cuda")
        self.k, self.v = (torch.zeros((layers, t, heads, dim), dtype=torch.float16, device="cuda") for _ in range(2))
        self.q = torch.zeros((layers, t, heads * group, dim), dtype=torch.float16, device="cuda")
        self.out = torch.full_like(self.q, 9.0)
        self.lse = torch.full((layers, t, heads * group), 9.0, device="cuda")

    def results(self):
        return [x.clone() for x in (self.starts, self.lengths, self.slots, self.positions, self.tables, self.out, self.lse)]

    def run(self, c, stream):
        c.plan(self.counts, self.tokens, self.most, rows=self.rows, starts=self.starts, lengths=self.lengths, slots=self.slots, positions=self.positions,
               tables=self.tables, stream=stream)
        for layer in range(len(self.k)):
            c.append(layer, self.k[layer], self.v[layer], stream=stream)
            c.attention(layer, self.q[layer], out=self.out[layer], lse=self.lse[layer], stream=stream)
        c.truncate(self.keep, rows=self.rows, stream=stream)


def inputs(step, seed, lengths, most):
    """Counts (0 for some), and how much of it all is kept, drawn on the CPU."""
    rng = np.random.default_rng(seed)
    rows = rng.permutation(step.n)
    counts = rng.integers(0, most + 1, step.n)
    keep = np.array([lengths[r] + rng.integers(0, c + 1) for r, c in zip(rows, counts)])
    for r, k in zip(rows, keep):
        lengths[r] = int(k)
    step.rows.copy_(ints(rows))
    step.counts.copy_(ints(counts))
    step.keep.copy_(ints(keep))
    for x in (step.k, step.v, step.q):
        x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float16)))
    step.out.fill_(9)
    step.lse.fill_(9)


@pytest.mark.parametrize("dim,group", [(128, 4), (64, 7)])
def test_captured_steps_share_a_cache(tq, dim, group):
    """Three graphs (prompts, drafts, single tokens) over one cache and its workspaces, replayed in turn with other counts, rows, values and lengths that
    the device holds: the same bits as the calls made one by one on another stream."""
    heads, n, layers, page = 2, 5, 2, 16
    eager_cache, graph_cache = (tq.PagedKVCache(layers, heads, dim, 130, page, n, 40, n * 100) for _ in range(2))
    mosts = [100, 6, 1]
    eager, captured = ([Step(n, m, heads, group, dim, layers) for m in mosts] for _ in range(2))
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for s in captured:          # counts of zero: nothing happens while warming up
        side.wait_stream(torch.cuda.current_stream())
        s.rows.copy_(torch.arange(n, dtype=torch.int32))
        torch.cuda.synchronize()
        s.run(graph_cache, side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            s.run(graph_cache, side)
            with pytest.raises(tq.TQError, match="captured plan"):
                graph_cache.plan(np.ones(1, np.int32), stream=side)
        graphs.append(g)
    lengths, same = [[0] * n, [0] * n], 0
    for turn, which in enumerate([0, 2, 1, 2, 1, 0, 1, 2, 2, 1]):
        for steps, held in ((eager, lengths[0]), (captured, lengths[1])):
            inputs(steps[which], turn, held, mosts[which])
        torch.cuda.synchronize()
        eager[which].run(eager_cache, other)
        graphs[which].replay()
        torch.cuda.synchronize()
        eager_cache.check_status()
        graph_cache.check_status()
        for a, b in zip(eager[which].results(), captured[which].results()):
            assert torch.equal(a, b), turn
            same += 1
        counted = int(captured[which].starts[-1])
        assert (captured[which].out[:, counted:] == 9).all() and torch.isfinite(captured[which].out[:, :counted].float()).all()
    assert same and eager_cache.free_pages() == graph_cache.free_pages() == 130 - sum(-(-x // page) for x in lengths[0])
    # a replay that does not fit says so and changes nothing
    captured[1].counts.fill_(7)
    before = graph_cache.free_pages()
    graphs[1].replay()
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="max_count"):
        graph_cache.check_status()
    assert graph_cache.free_pages() == before
    eager_cache.close()
    graph_cache.close()


def test_caches_side_by_side(tq):
    """Two caches on two streams at once, with both kernels at work: each as if it were alone."""
    torch.manual_seed(3)
    streams = [torch.cuda.Stream() for _ in range(2)]
    data = [[torch.randn((s, h, 128), device="cuda").half() for s, h in ((1212, 2), (1212, 2), (1212, 8))] for _ in range(2)]
    counts = np.array([1, 1, 10, 1200], np.int32)

    def make():
        return tq.PagedKVCache(1, 2, 128, 200, 64, 4, 200, 1212)

    def steps(c, x, stream, times):
        out = []
        for _ in range(times):
            c.plan(counts, stream=stream)
            c.append(0, x[0], x[1], stream=stream)
            out.append(torch.empty_like(x[2]))
            with torch.cuda.stream(stream):
                out[-1].zero_()
            c.attention(0, x[2], out=out[-1], stream=stream)
        return out

    alone = []
    for x, s in zip(data, streams):
        c = make()
        torch.cuda.synchronize()
        alone.append(steps(c, x, s, 4))
        torch.cuda.synchronize()
        c.check_status()
        c.close()
    caches = [make() for _ in range(2)]
    torch.cuda.synchronize()
    together = [[], []]
    for _ in range(4):
        for i in range(2):
            together[i] += steps(caches[i], data[i], streams[i], 1)
    torch.cuda.synchronize()
    for c in caches:
        c.check_status()
    for a, b in zip(alone, together):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for c in caches:
        c.close()


@pytest.mark.parametrize("handle", [False, True])
def test_results_without_a_place_on_another_stream(tq, handle):
    """The zeros that attention makes room with are in front of it, whatever the current stream has to do first."""
    c = tq.PagedKVCache(1, 2, 128, 8, 64, 2, 8, 40)
    x = torch.randn((40, 2, 128), device="cuda").half()
    c.plan(np.array([5, 30], np.int32), 40, 30)
    c.append(0, x, x)
    want = c.attention(0, x)
    big = torch.randn((6000, 6000), device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(4):
        big = big @ big * 1e-4
    out = c.attention(0, x, stream=side.cuda_stream if handle else side)
    torch.cuda.synchronize()
    c.check_status()
    assert torch.equal(out, want) and (want[:35] != 0).any() and (want[35:] == 0).all()
    with torch.cuda.stream(side):          # (no stream named: the default one)
        for _ in range(4):
            big = big @ big * 1e-4
        out = c.attention(0, x)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    c.close()
