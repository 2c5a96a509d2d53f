"""What the paged cache's Python calls hand on: numbers that fit, in front of the C interface, which takes 32 bits of any."""
import ctypes

import numpy as np
import pytest

import turboquant_mlx_core_b200 as tq
from turboquant_mlx_core_b200 import paged

torch = pytest.importorskip("torch")


class Library:
    """Takes every call down."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def cache():
    paged._load_torch()
    c = object.__new__(tq.PagedKVCache)
    c._L, c._h = Library(), 1
    c.num_layers, c.num_heads, c.head_dim, c.page_tokens, c.max_tokens = 1, 2, 64, 16, 100
    yield c
    c._h = None


def numbers(call, n):
    """The n numbers at an address that was handed on."""
    return np.ctypeslib.as_array((ctypes.c_int32 * n).from_address(call)).tolist()


@pytest.mark.parametrize("counts", [[3, 0, 5], (3, 0, 5), np.array([3, 0, 5]), np.array([3, 0, 5], np.uint8), np.array([3, 9, 0, 9, 5], np.int32)[::2], np.array([3, 0, 5], np.uint64)])
def test_whole_numbers_of_any_kind(cache, counts, monkeypatch):
    seen = []
    monkeypatch.setattr(cache._L, "tq_paged_plan", lambda *a: seen.append((a[3:6], numbers(a[2], 3))) or 0, raising=False)
    monkeypatch.setattr(cache._L, "tq_paged_truncate", lambda *a: seen.append(numbers(a[2], 3)) or 0, raising=False)
    cache.plan(counts)
    cache.truncate(counts)
    assert seen == [((3, 8, 5), [3, 0, 5]), [3, 0, 5]]


@pytest.mark.parametrize("bad,error", [(np.array([2 ** 32 + 3]), ValueError), (np.array([-2 ** 31 - 1]), ValueError), (np.array([2 ** 64 - 1], np.uint64), ValueError),
                                       ([2 ** 31], ValueError), (np.array([1.0]), TypeError), ([1.5], TypeError), (np.array([True]), TypeError)])
def test_numbers_that_do_not_fit(cache, bad, error):
    for call in (lambda: cache.plan(bad), lambda: cache.plan(bad, 8, 8), lambda: cache.truncate(bad)):
        with pytest.raises(error, match="counts|lengths"):
            call()
    assert cache._L.calls == []


@pytest.mark.parametrize("wide", [2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 31 - 1, 2 ** 64])
def test_arguments_that_do_not_fit(cache, wide):
    one, x = np.ones(1, np.int32), torch.zeros((3, 2, 64), dtype=torch.float16)
    calls = [lambda: cache.plan(one, wide, 1), lambda: cache.plan(one, 1, wide), lambda: cache.append(wide, x, x), lambda: cache.attention(wide, x, out=x),
             lambda: cache.attention(0, x, out=x, window=wide), lambda: cache.read_pages(wide, torch.zeros(1, dtype=torch.int32)),
             lambda: tq.PagedKVCache(1, 2, 64, wide), lambda: tq.PagedKVCache(1, 2, 64, 4, max_tokens=wide), lambda: tq.PagedKVCache(wide, 2, 64, 4)]
    for call in calls:
        with pytest.raises(ValueError, match="32 bits"):
            call()
    assert cache._L.calls == []


def test_a_sum_of_counts_that_does_not_fit(cache):
    with pytest.raises(ValueError, match="32 bits"):
        cache.plan(np.array([2 ** 31 - 1, 2 ** 31 - 1, 3], np.int32))       # (2^32 + 1)
    assert cache._L.calls == []


def test_no_counts(cache):
    for empty in ([], np.zeros(0), np.zeros(0, np.int32)):
        cache.plan(empty)
        assert cache._L.calls[-1][0] == "tq_paged_plan" and cache._L.calls[-1][1][3:6] == (0, 0, 0)
