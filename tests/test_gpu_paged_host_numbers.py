"""GPU tests of rows, counts and lengths in host memory: a call has read them when it returns, from whatever memory."""
import numpy as np
import pytest

from tests.paged_model import Model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def busy(stream):
    """Some tens of milliseconds of work, so that what is queued behind is read late if it is not read at once."""
    with torch.cuda.stream(stream):
        big = torch.ones((8192, 8192), device="cuda")
        for _ in range(8):
            big = big @ big * 1e-4
    return big


def host(kind, n):
    """An array of n numbers and the same memory as numpy."""
    x = torch.zeros(n, dtype=torch.int32, pin_memory=kind != "pageable")
    return (x if kind == "pinned tensor" else x.numpy()), x.numpy()


@pytest.mark.parametrize("kind", ["pageable", "pinned tensor", "pinned numpy"])
@pytest.mark.parametrize("n", [3, 1000])
def test_numbers_are_read_before_a_call_returns(tq, kind, n):
    """One buffer for each of rows, counts and lengths, filled anew for every call while the device is behind."""
    c = tq.PagedKVCache(1, 1, 64, 40 * n, 16, n, 40, 20 * n)
    m = Model(1, 64, 1, 16)
    m.stack = list(range(40 * n))[::-1]
    (rows, set_rows), (counts, set_counts), (lengths, set_lengths) = (host(kind, n) for _ in range(3))
    rng = np.random.default_rng(n)
    stream = torch.cuda.Stream()
    got, want = [], []
    for step in range(4):
        kept = busy(stream)
        set_rows[:] = rng.permutation(n)
        set_counts[:] = rng.integers(0, 20, n)
        out = {"starts": torch.full((n + 1,), 77, dtype=torch.int32, device="cuda"), "slots": torch.full((20 * n,), 77, dtype=torch.int32, device="cuda")}
        torch.cuda.current_stream().synchronize()
        slots, _ = m.plan(set_counts.tolist(), set_rows.tolist())
        want.append(([0, *np.cumsum(set_counts)], slots + [-1] * (20 * n - len(slots))))
        c.plan(counts, 20 * n, 20, rows=rows, stream=stream, **out)
        got.append(out)
        set_counts[:] = 1
        set_rows[:] = set_rows[::-1].copy()
        keep = [int(rng.integers(0, m.lengths[r] + 1)) for r in set_rows]
        set_lengths[:] = keep
        m.truncate(keep, set_rows.tolist())
        c.truncate(lengths, rows=rows, stream=stream)
        set_lengths[:] = 0
        set_rows[:] = -1
        del kept
    torch.cuda.synchronize()
    c.check_status()
    for out, (starts, slots) in zip(got, want):
        assert out["starts"].tolist() == starts and out["slots"].tolist() == slots
    assert c.free_pages() == len(m.stack)
    c.close()
