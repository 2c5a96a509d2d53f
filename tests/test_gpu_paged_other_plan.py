"""GPU tests of appends and attentions that find another plan on the device than the one that they were made for: a captured step was
replayed, or a truncation, between the plan and the call."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DIM, HEADS, GROUP = 64, 2, 2


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def rows(tokens, heads=HEADS):
    return torch.randn((tokens, heads, DIM), device="cuda").half()


class Captured:
    """A step of requests 4 .. of `counts` tokens each as a graph that holds its plan, its append, its attention and its truncation."""

    def __init__(self, c, counts, truncate=False):
        self.counts, self.rows, self.keep = ints(counts), ints(range(4, 4 + len(counts))), ints([0] * len(counts))
        tokens, most = sum(counts), max(counts)
        k, q = rows(tokens), rows(tokens, HEADS * GROUP)
        out = torch.empty_like(q)
        side = torch.cuda.Stream()
        self.graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(self.graph, stream=side):
            c.plan(self.counts, tokens, most, rows=self.rows, stream=side)
            c.append(0, k, k, stream=side)
            c.attention(0, q, out=out, stream=side)
            if truncate:
                c.truncate(self.keep, rows=self.rows, stream=side)
        self.held = (k, q, out)


def pages_of(c):
    out = [torch.empty((c.num_pages, c.page_tokens, HEADS, DIM), device="cuda") for _ in range(2)]
    c.read_pages(0, ints(range(c.num_pages)), *out)
    return out


# (counts of the plan, counts of the captured step)
SIZES = [([1, 1], [1, 1, 1]), ([1, 1, 1], [1, 1]), ([1, 1], [5, 3]), ([3, 2], [1, 1]), ([8, 8], [12, 4]), ([2, 2], [40, 30]), ([40, 30], [1, 1]), ([70], [70, 70]), ([1], [100])]


@pytest.mark.parametrize("mine,other", SIZES)
@pytest.mark.parametrize("truncate", [False, True])
def test_a_replay_between_a_plan_and_its_calls(tq, mine, other, truncate):
    c = tq.PagedKVCache(1, HEADS, DIM, 60, 16, 8, 12, 200)
    step = Captured(c, other, truncate)
    c.plan(np.array([20, 30], np.int32))
    x = rows(50)
    c.append(0, x, x)
    tokens = sum(mine)
    k, q = rows(tokens), rows(tokens, HEADS * GROUP)
    c.plan(np.array(mine, np.int32))
    torch.cuda.synchronize()
    c.check_status()
    step.graph.replay()
    torch.cuda.synchronize()
    c.check_status()
    before, free = pages_of(c), c.free_pages()
    out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda")
    for call in (lambda: c.append(0, k, k), lambda: c.attention(0, q, out=out, lse=lse)):
        call()
        torch.cuda.synchronize()
        with pytest.raises(tq.TQError, match="not the one"):
            c.check_status()
        c.check_status()
    assert (out == 9).all() and (lse == 9).all() and c.free_pages() == free
    assert all(torch.equal(a, b) for a, b in zip(before, pages_of(c)))
    # a plan of its own sets it right
    c.plan(np.array(mine, np.int32))
    c.append(0, k, k)
    c.attention(0, q, out=out, lse=lse)
    torch.cuda.synchronize()
    c.check_status()
    assert torch.isfinite(out).all() and not (lse == 9).any()
    c.close()


def test_a_replayed_truncation_ends_the_plan(tq):
    c = tq.PagedKVCache(1, HEADS, DIM, 20, 16, 4, 8, 100)
    keep, which = ints([3]), ints([1])
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        c.truncate(keep, rows=which, stream=side)
    c.plan(np.array([6, 5], np.int32))
    graph.replay()
    x = rows(11)
    out = torch.full_like(x, 9.0)
    c.append(0, x, x)
    c.attention(0, x, out=out)
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="not the one"):
        c.check_status()
    assert (out == 9).all()
    c.close()


def test_a_plan_that_was_refused_says_why(tq):
    """(and not that it is another)"""
    c = tq.PagedKVCache(1, HEADS, DIM, 3, 16, 4, 8, 100)
    c.plan(np.array([60, 20], np.int32))
    x = rows(80)
    out = torch.full_like(x, 9.0)
    c.append(0, x, x)
    c.attention(0, x, out=out)
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="free pages"):
        c.check_status()
    assert (out == 9).all()
    c.close()
