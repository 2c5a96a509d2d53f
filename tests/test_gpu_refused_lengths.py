"""GPU tests of the lengths that a refused plan and a kept branch behind it give: what the requests hold."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("rows,counts,want", [
    ([0, 1, 2], [3, 9, 2], [20, 10, 5]),                # a count above max_count
    ([0, 1, 2], [3, -1, 2], [20, 10, 5]),
    ([2, 1, 0], [8, 8, 8], [5, 10, 20]),                # more tokens than announced
    ([0, 1, 1], [3, 2, 2], [20, 10, 10]),               # a row named twice
    ([1, 1, 1], [3, 9, -2], [10, 10, 10]),
    ([0, 3, 2], [3, 2, 2], [20, 0, 5]),                 # rows outside the tables
    ([0, -1, 1 << 30], [3, 2, 2], [20, 0, 0]),
    ([0, 1, 2], [7, 0, 0], [20, 10, 5]),                # longer than a row of the tables
])
def test_lengths_behind_a_refused_plan(tq, rows, counts, want):
    long = counts == [7, 0, 0]
    c = tq.PagedKVCache(1, 1, 64, 12, 16, 3, 2 if long else 4, 64)
    c.plan(np.array([20, 10, 5], np.int32))
    if long:
        c.plan(np.array([6, 0, 0], np.int32))
        want = [26, 10, 5]
    free = c.free_pages()
    lengths, kept, tables = (torch.full(s, 77, dtype=torch.int32, device="cuda") for s in ((3,), (3,), (3, 4)))
    c.plan(ints(counts), 16, 8, rows=ints(rows), lengths=lengths, tables=tables)
    c.keep(ints([[0], [0], [0]]), ints([1, 1, 1]), lengths=kept)
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="row|count|longer|tokens"):
        c.check_status()
    assert lengths.tolist() == want and kept.tolist() == want
    assert [(t >= 0).sum().item() for t in tables] == [-(-n // 16) for n in want]
    assert c.free_pages() == free
    c.check_status()
    # nothing has changed: the same rows go on from there
    positions = torch.zeros(3, dtype=torch.int32, device="cuda")
    c.plan(np.array([1, 1, 1], np.int32), positions=positions)
    assert positions.tolist() == [26 if long else 20, 10, 5]
    c.check_status()
    c.close()


def test_a_replayed_plan_that_is_refused(tq):
    """A loop on the device goes by the lengths: a plan and a keep in a graph, with counts that fit and that do not."""
    c = tq.PagedKVCache(1, 1, 64, 12, 16, 2, 6, 64)
    c.plan(np.array([20, 10], np.int32))
    counts, path, kept, lengths = ints([0, 0]), ints([[0, 1], [0, 1]]), ints([0, 0]), ints([77, 77])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.plan(counts, 8, 4, stream=side)
            c.keep(path, kept, lengths=lengths, stream=side)
    for new, stay, want in (([4, 4], [2, 1], [22, 11]), ([5, 4], [2, 1], [22, 11]), ([1, -1], [1, 0], [22, 11]), ([1, 2], [1, 2], [23, 13])):
        counts.copy_(ints(new))
        kept.copy_(ints(stay))
        graph.replay()
        torch.cuda.synchronize()
        assert lengths.tolist() == want
        if max(new) > 4 or min(new) < 0:
            with pytest.raises(tq.TQError, match="count"):
                c.check_status()
        else:
            c.check_status()
    c.close()
