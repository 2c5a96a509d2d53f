"""The paged cache's calls that are refused before any device work."""
import numpy as np
import pytest

import turboquant_mlx_core_b200 as tq
from tests.paged_model import FLOOR, Model, exponent


@pytest.mark.parametrize("change,what", [
    ({"num_layers": 0}, "positive"), ({"num_heads": 0}, "positive"), ({"num_pages": -1}, "positive"), ({"head_dim": 96}, "head_dim"),
    ({"page_tokens": 48}, "page"), ({"page_tokens": 256}, "page"), ({"max_requests": 0}, "max_requests"), ({"max_requests": 4097}, "max_requests"),
    ({"max_pages_per_request": 0}, "positive"), ({"max_tokens": 0}, "positive"), ({"num_pages": 1 << 24, "page_tokens": 128}, "tokens"),
    ({"num_pages": 1 << 23, "num_heads": 256}, "pages times heads"), ({"num_pages": 1, "num_heads": 65537}, "65536 heads")])
def test_caches_that_cannot_be(change, what):
    sizes = dict(num_layers=1, num_heads=2, head_dim=128, num_pages=4, page_tokens=64, max_requests=2, max_pages_per_request=4, max_tokens=8)
    with pytest.raises(tq.TQError, match=what):
        tq.PagedKVCache(**{**sizes, **change})


def test_null_handles():
    L = tq.load()
    L.tq_paged_cache_free(None)
    one = np.ones(1, np.int32)
    for rc in (L.tq_paged_plan(None, None, one.ctypes.data, 1, 1, 1, None, None, None, None, None, 0, None),
               L.tq_paged_truncate(None, None, one.ctypes.data, 1, None), L.tq_paged_append(None, 0, None, None, 1, 1, 256, 256, None),
               L.tq_paged_read(None, 0, None, 1, None, None, 1, None),
               L.tq_paged_attention(None, 0, None, 1, 2, 256, 0, 0.0, None, 256, None, None), L.tq_paged_status(None)):
        assert rc != 0 and b"NULL" in L.tq_last_error()
    assert L.tq_paged_free_pages(None) == -1


def test_exponents():
    """The least power of two: a code of 127 is reached from 126.5 on, and 127.5 takes the next one."""
    assert exponent(0.0) == FLOOR and exponent(2.0 ** -140) == FLOOR and exponent(np.inf) is None and exponent(np.nan) is None
    for e in (-24, -3, 0, 5, 100):
        assert exponent(127 * 2.0 ** e) == e and exponent(127.4999 * 2.0 ** e) == e and exponent(127.5 * 2.0 ** e) == e + 1
        assert exponent(63.75 * 2.0 ** e) == e and exponent(63.7499 * 2.0 ** e) == e - 1


def test_model_takes_pages_back_in_order():
    m = Model(1, 64, 12, 16)
    m.plan([20, 33, 0])
    first = {r: list(t) for r, t in m.tables.items()}
    stack = list(m.stack)
    m.plan([30, 1, 50])
    grown = {r: list(t) for r, t in m.tables.items()}
    m.truncate([20, 33, 0])
    assert m.tables == first and m.stack == stack
    m.plan([30, 1, 50])
    assert m.tables == grown
