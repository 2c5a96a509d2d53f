"""GPU tests of a tree that is replayed behind a plan of other sizes: nothing of it is done, its positions are as they were."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("chains", [True, False])
@pytest.mark.parametrize("other", ["plan", "truncate", "keep"])
def test_positions_behind_another_plan(tq, other, chains):
    c = tq.PagedKVCache(1, 1, 64, 20, 16, 2, 10, 64)
    c.plan(np.array([20, 10], np.int32))
    parents, positions = None if chains else ints([-1, 0, 0, -1, 0, 1]), torch.full((6,), 9, dtype=torch.int32, device="cuda")
    queries = torch.ones((6, 1, 64), dtype=torch.float16, device="cuda")
    out = torch.full_like(queries, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.plan(ints([3, 3]), 6, 3, stream=side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.tree(parents, positions=positions, stream=side)
            c.tree_attention(0, queries, out=out, stream=side)
        if other == "plan":
            c.plan(ints([1]), 1, 1, stream=side)
        elif other == "truncate":
            c.truncate(ints([20, 10]), stream=side)
        else:
            c.keep(ints([[0], [0]]), ints([1, 1]), stream=side)
        graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="plan on the device"):
        c.check_status()
    assert positions.tolist() == [9] * 6 and (out == 9).all()
    # behind a plan of these sizes it is done, and a refused one has no tokens
    with torch.cuda.stream(side):
        c.plan(ints([3, 1]), 6, 3, stream=side)
        graph.replay()
    torch.cuda.synchronize()
    c.check_status()
    held = {"plan": [24, 13], "truncate": [20, 10], "keep": [21, 11]}[other]
    assert positions.tolist() == [held[0] + d for d in ((0, 1, 2) if chains else (0, 1, 1))] + [held[1], 0, 0]
    with torch.cuda.stream(side):
        c.plan(ints([4, 1]), 6, 3, stream=side)
        graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(tq.TQError, match="count"):
        c.check_status()
    assert positions.tolist() == [0] * 6
    c.close()
