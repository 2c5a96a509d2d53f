"""GPU tests of trees of drafts in the paged cache: positions, and kept branches, against their definitions."""
import numpy as np
import pytest

from tests import drafts_model
from tests.paged_model import Model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def paths_tensor(paths, width):
    return ints([(list(p or []) + [-1] * width)[:width] for p in paths])


class Pair:
    """A cache of some layers and its models."""

    def __init__(self, tq, heads, dim, page, requests, pages, layers=1, max_tokens=4096):
        self.c = tq.PagedKVCache(layers, heads, dim, pages, page, requests, pages, max_tokens)
        self.m = [Model(heads, dim, pages, page) for _ in range(layers)]
        self.shape = (heads, dim)

    def step(self, rng, counts, rows, spread=1.0, keys=None):
        for m in self.m:
            m.plan(counts, rows)
        self.c.plan(np.array(counts, np.int32), rows=ints(rows))
        for i, m in enumerate(self.m):
            kv = [(rng.standard_normal((sum(counts), *self.shape)) * np.exp(spread * rng.standard_normal((sum(counts), 1, 1)))).astype(np.float16) for _ in range(2)]
            if keys is not None:
                kv[0] = keys
            for which, x in enumerate(kv):
                m.append(which, x)
            if sum(counts):
                self.c.append(i, *(torch.from_numpy(x).cuda() for x in kv))

    def keep(self, paths, rows, width=None):
        width = width or max(1, *(len(p or []) for p in paths))
        lengths = torch.full((len(paths),), 77, dtype=torch.int32, device="cuda")
        self.c.keep(paths_tensor(paths, width), ints([-1 if p is None else len(p) for p in paths]), lengths=lengths)
        for m in self.m:
            for which in (0, 1):
                drafts_model.keep(m, which, paths)
        want = drafts_model.kept_lengths(self.m[0], paths)
        for m in self.m:
            m.truncate(want, rows)
        assert lengths.tolist() == want

    def compare(self, pages):
        """All pages, whatever they hold."""
        page, (heads, dim) = self.c.page_tokens, self.shape
        for i, m in enumerate(self.m):
            got = [torch.empty((pages, page, heads, dim), device="cuda") for _ in range(2)]
            self.c.read_pages(i, ints(range(pages)), *got)
            for which in (0, 1):
                assert np.array_equal(got[which].cpu().numpy().astype(np.float64), m.values(which, range(pages)), equal_nan=True), f"layer {i}, {which}"
        torch.cuda.synchronize()
        self.c.check_status()
        assert self.c.free_pages() == len(self.m[0].stack)


@pytest.mark.parametrize("spread", [0, 1, 2, 8, 300])
def test_positions_of_trees(tq, spread):
    rng = np.random.default_rng(spread)
    counts = [1, 7, 0, 64, 256, 31, 2, 255]
    p = Pair(tq, 1, 64, 16, 8, 200)
    p.step(rng, [5, 0, 3, 100, 16, 15, 0, 1], range(8))
    p.c.plan(np.array(counts, np.int32), tokens=sum(counts) + 3)
    parents = drafts_model.trees(rng, counts, spread)
    positions = torch.full((sum(counts) + 3,), 77, dtype=torch.int32, device="cuda")
    p.c.tree(ints(np.concatenate([np.asarray(x, np.int32) for x in parents] + [np.full(3, -9, np.int32)])), positions=positions)
    want = [h + d for h, par in zip([5, 0, 3, 100, 16, 15, 0, 1], parents) for d in drafts_model.depths(par)] + [0] * 3
    assert positions.tolist() == want
    torch.cuda.synchronize()
    p.c.check_status()
    p.c.close()


def test_long_chains_and_forests(tq):
    p = Pair(tq, 1, 64, 16, 3, 200)
    counts = [1000, 4, 300]
    p.c.plan(np.array(counts, np.int32))
    positions = torch.zeros(1304, dtype=torch.int32, device="cuda")
    p.c.tree(None, positions=positions)
    assert positions.tolist() == [*range(1000), *range(4), *range(300)]
    p.c.tree(ints([*range(-1, 999), -1, -1, 1, -1, *range(-1, 299)]), positions=positions)
    assert positions.tolist() == [*range(1000), 0, 0, 1, 0, *range(300)]
    p.c.tree()
    torch.cuda.synchronize()
    p.c.check_status()
    p.c.close()


@pytest.mark.parametrize("bad", [0, 1, 5, -2, 1 << 30, -(1 << 31)])
def test_parents_that_make_no_tree(tq, bad):
    """Of the request whose parents they are alone."""
    p = Pair(tq, 1, 64, 16, 3, 200)
    p.c.plan(np.array([3, 4, 300], np.int32))
    parents, positions = [-1, 0, 0, -1, bad, 0, 1, -1, *range(299)], torch.zeros(307, dtype=torch.int32, device="cuda")
    if bad == 0:
        parents[10] = 0          # 300 nodes that are no chain
        parents[4] = 3           # (itself would be 1: 3 is behind it)
    p.c.tree(ints(parents), positions=positions)
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="tree"):
        p.c.check_status()
    got = positions.tolist()
    assert got[:3] == [0, 1, 1] and got[3:7] == [0] * 4 and got[7:] == ([0] * 300 if bad == 0 else list(range(300)))
    p.c.check_status()
    p.c.close()


def random_paths(rng, parents):
    paths = []
    for par in parents:
        if not par or rng.random() < 0.15:
            paths.append([] if rng.random() < 0.5 else None)
            continue
        j, path = int(rng.integers(len(par))), []
        while j >= 0:
            path.append(j)
            j = par[j]
        paths.append(path[::-1])
    return paths


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,layers", [(1, 1), (3, 2)])
def test_kept_branches(tq, dim, page, heads, layers):
    """Several steps of trees, of which a branch each stays; every page's numbers, free pages and lengths after each."""
    rng = np.random.default_rng(dim + page + heads)
    n, pages = 7, 90
    p = Pair(tq, heads, dim, page, n, pages, layers)
    rows = rng.permutation(n).tolist()
    p.step(rng, [0, 3, 15, 16, page - 1, page, 77], rows)
    for turn in range(4):
        counts = [int(rng.integers(0, 70)) for _ in range(n)]
        parents = drafts_model.trees(rng, counts, [1, 3, 12, 40][turn])
        p.step(rng, counts, rows, spread=1.5)
        p.c.tree(ints(np.concatenate([np.asarray(x, np.int32) for x in parents])))
        p.keep(random_paths(rng, parents), rows)
        p.compare(pages)
    p.c.close()


@pytest.mark.parametrize("page", [16, 64])
def test_any_ascending_list_may_stay(tq, page):
    rng = np.random.default_rng(page)
    n, pages = 4, 120
    p = Pair(tq, 2, 64, page, n, pages)
    rows = list(range(n))
    p.step(rng, [9, 0, 40, 16], rows)
    for share in (0.1, 0.5, 0.9, 1.0):
        counts = [200, 33, 1, 90]
        p.step(rng, counts, rows, spread=2.0)
        paths = [np.nonzero(rng.random(c) < share)[0].tolist() for c in counts]
        p.keep(paths, rows, width=201)
        p.compare(pages)
    p.c.close()


def test_pages_that_are_not_numbers(tq):
    rng = np.random.default_rng(3)
    p = Pair(tq, 2, 64, 16, 3, 40)
    rows = [0, 1, 2]
    p.step(rng, [10, 14, 2], rows)
    keys = rng.standard_normal((60, 2, 64)).astype(np.float16)
    keys[18, 0, 5] = np.nan      # a page behind request 0's first one
    keys[22, 1, 0] = np.inf      # request 1's first one
    p.step(rng, [20, 20, 20], rows, keys=keys)
    p.keep([[0, 8, 19], [1, 5, 6, 7], [3, 19]], rows)
    p.compare(40)
    p.c.close()


def test_all_and_none_stay(tq):
    rng = np.random.default_rng(4)
    p = Pair(tq, 1, 128, 32, 3, 40)
    p.step(rng, [31, 0, 5], [0, 1, 2])
    p.step(rng, [40, 33, 1], [0, 1, 2])
    p.keep([None, [], list(range(1))], [0, 1, 2], width=1)
    p.compare(40)
    p.c.close()


@pytest.mark.parametrize("path,kept", [([0, 5], 2), ([3, 2], 2), ([1, 1], 2), ([-1, 2], 2), ([0, 1], 3), ([0, 1 << 30], 2), ([0, 1], 1 << 30)])
def test_paths_that_are_none_change_nothing(tq, path, kept):
    rng = np.random.default_rng(5)
    p = Pair(tq, 1, 64, 16, 2, 20)
    p.step(rng, [20, 20], [0, 1])
    p.step(rng, [5, 5], [0, 1])
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    p.c.keep(ints([[0, 3], path]), ints([2, kept]), lengths=lengths)
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="path"):
        p.c.check_status()
    assert lengths.tolist() == [25, 25]
    p.compare(20)
    with pytest.raises(tq.TQError, match="no plan"):
        p.c.keep(ints([[0], [0]]), ints([1, 1]))
    p.c.close()


def test_calls_out_of_turn(tq):
    p = Pair(tq, 1, 64, 16, 2, 20)
    one, path = ints([0]), ints([[0]])
    for call in (lambda: p.c.tree(one), lambda: p.c.keep(path, one)):
        with pytest.raises(tq.TQError, match="no plan"):
            call()
    p.c.plan(np.array([3, 2], np.int32))
    for call in (lambda: p.c.tree(ints([0] * 4)), lambda: p.c.keep(path, one), lambda: p.c.tree(torch.zeros(5, dtype=torch.int32)),
                 lambda: p.c.keep(torch.zeros((2, 1), dtype=torch.int32), ints([0, 0]))):
        with pytest.raises(tq.TQError):
            call()
    p.c.close()


def test_a_refused_plan_keeps_nothing(tq):
    rng = np.random.default_rng(6)
    p = Pair(tq, 1, 64, 16, 2, 4)
    p.step(rng, [20, 10], [0, 1])
    p.c.plan(ints([40, 1]), 41, 40)       # no pages left
    positions = torch.full((41,), 5, dtype=torch.int32, device="cuda")
    p.c.tree(None, positions=positions)
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    p.c.keep(ints([[0], [0]]), ints([1, 1]), lengths=lengths)
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="free pages"):
        p.c.check_status()
    assert lengths.tolist() == [20, 10] and positions.tolist() == [0] * 41
    p.compare(4)
    p.c.close()


def test_another_plan_on_the_device(tq):
    """A captured step's plan, tree and kept branch behind a plan of other sizes: nothing is done, and the status tells."""
    rng = np.random.default_rng(7)
    p = Pair(tq, 1, 64, 16, 2, 20)
    p.step(rng, [20, 10], [0, 1])
    counts, path, kept, lengths = ints([3, 3]), ints([[0, 2], [1, 2]]), ints([2, 2]), torch.full((2,), 9, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.c.plan(counts, 6, 3, stream=side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            p.c.keep(path, kept, lengths=lengths, stream=side)
        p.c.plan(ints([1]), 1, 1, stream=side)
        graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="plan on the device"):
        p.c.check_status()
    assert lengths.tolist() == [9, 9]
    p.c.close()


def test_a_captured_step(tq):
    """Plan, tree, append and keep in a graph, replayed with other trees, paths and lengths than at its capture."""
    rng = np.random.default_rng(8)
    n, most, pages = 5, 12, 60
    p = Pair(tq, 2, 64, 16, n, pages, 2)
    rows = list(range(n))
    p.step(rng, [20, 1, 15, 0, 33], rows)
    counts, parents = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n * most, dtype=torch.int32, device="cuda")
    path, kept, lengths = torch.zeros((n, most), dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    positions = torch.zeros(n * most, dtype=torch.int32, device="cuda")
    kv = [[torch.zeros((n * most, 2, 64), dtype=torch.float16, device="cuda") for _ in range(2)] for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        p.c.plan(counts, n * most, most, stream=side)
        p.c.tree(parents, positions=positions, stream=side)
        for i in range(2):
            p.c.append(i, *kv[i], stream=side)
        p.c.keep(path, kept, lengths=lengths, stream=side)

    with torch.cuda.stream(side):
        step()          # (no tokens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for _ in range(5):
        c = [int(rng.integers(0, most + 1)) for _ in range(n)]
        trees = drafts_model.trees(rng, c, 4)
        paths = [p_ or [] for p_ in random_paths(rng, trees)]
        counts.copy_(ints(c))
        parents.fill_(-5)
        parents[:sum(c)] = ints(np.concatenate([np.asarray(t, np.int32) for t in trees])) if sum(c) else parents[:0]
        path.copy_(paths_tensor(paths, most))
        kept.copy_(ints([len(x) for x in paths]))
        held = [p.m[0].lengths.get(r, 0) for r in rows]
        for i, m in enumerate(p.m):
            m.plan(c, rows)
            for which in (0, 1):
                x = rng.standard_normal((sum(c), 2, 64)).astype(np.float16)
                m.append(which, x)
                kv[i][which][:sum(c)] = torch.from_numpy(x).cuda()
        graph.replay()
        torch.cuda.synchronize()
        assert positions.tolist()[:sum(c)] == [h + d for h, t in zip(held, trees) for d in drafts_model.depths(t)]
        for m in p.m:
            for which in (0, 1):
                drafts_model.keep(m, which, paths)
        want = drafts_model.kept_lengths(p.m[0], paths)
        for m in p.m:
            m.truncate(want, rows)
        assert lengths.tolist() == want
        p.compare(pages)
    p.c.close()


def test_a_branch_is_kept_once(tq):
    """A captured keep that is replayed again without a plan moves nothing more, and the status tells."""
    rng = np.random.default_rng(9)
    p = Pair(tq, 2, 64, 16, 2, 20)
    p.step(rng, [20, 10], [0, 1])
    path, kept, lengths = ints([[1, 3, 4], [0, 2, -1]]), ints([3, 2]), torch.full((2,), 9, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    p.step(rng, [5, 5], [0, 1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        p.c.keep(path, kept, lengths=lengths, stream=side)
    graph.replay()
    for m in p.m:
        for which in (0, 1):
            drafts_model.keep(m, which, [[1, 3, 4], [0, 2]])
        m.truncate([23, 12], [0, 1])
    assert lengths.tolist() == [23, 12]
    p.compare(20)
    for _ in range(2):
        lengths.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        with pytest.raises(tq.TQError, match="plan on the device"):
            p.c.check_status()
        assert lengths.tolist() == [9, 9]
        p.compare(20)
    p.c.close()


def test_results_where_the_paths_are(tq):
    """Refused: the moves read the paths and their lengths behind the bookkeeping.  Next to them they may be."""
    rng = np.random.default_rng(10)
    p = Pair(tq, 1, 64, 16, 2, 20)
    p.step(rng, [20, 10], [0, 1])
    p.step(rng, [5, 5], [0, 1])
    block = ints([0, 4, 1, 2, 2, 2, 77, 77])
    path, kept = block[:4].view(2, 2), block[4:6]
    for lengths in (kept, block[5:7], block[3:5], block[:2]):
        with pytest.raises(tq.TQError, match="must not be where"):
            p.c.keep(path, kept, lengths=lengths)
    p.c.keep(path, kept, lengths=block[6:])
    for which in (0, 1):
        drafts_model.keep(p.m[0], which, [[0, 4], [1, 2]])
    p.m[0].truncate([22, 12], [0, 1])
    assert block.tolist() == [0, 4, 1, 2, 2, 2, 22, 12]
    p.compare(20)
    p.c.close()


def test_paths_in_wide_rows(tq):
    """A path's row may be longer than any request's new tokens; what is behind it is not looked at."""
    rng = np.random.default_rng(11)
    p = Pair(tq, 1, 64, 16, 2, 20)
    p.step(rng, [20, 10], [0, 1])
    p.step(rng, [5, 3], [0, 1])
    path = torch.full((2, 70000), 1 << 30, dtype=torch.int32, device="cuda")
    path[0, :2], path[1, :3] = ints([2, 4]), ints([0, 1, 2])
    p.c.keep(path, ints([2, 3]))
    for which in (0, 1):
        drafts_model.keep(p.m[0], which, [[2, 4], [0, 1, 2]])
    p.m[0].truncate([22, 13], [0, 1])
    p.compare(20)
    p.c.close()
