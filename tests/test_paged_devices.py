"""Tensors of another device than the cache's are refused in front of the C interface: a kernel that reads them would fault."""
import pytest

from tests.test_paged_arguments import cache  # noqa: F401

torch = pytest.importorskip("torch")


class Elsewhere:
    """A tensor of another device."""
    is_cuda = True

    def __init__(self, x, device=1):
        self.x, self.device_index = x, device

    def get_device(self):
        return self.device_index

    def __getattr__(self, name):
        return getattr(self.x, name)


def test_tensors_of_another_device(cache):  # noqa: F811
    cache._device = 0
    x, n = torch.zeros((3, 2, 64), dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    pages = torch.zeros((3, 16, 2, 64), dtype=torch.float16)
    here, there = (lambda t: Elsewhere(t, 0)), Elsewhere
    calls = [lambda f: cache.plan(f(n), 3, 1), lambda f: cache.plan(n, 3, 1, rows=f(n)), lambda f: cache.plan(n, 3, 1, slots=f(n)), lambda f: cache.plan(n, 3, 1, lengths=f(n)),
             lambda f: cache.plan(n, 3, 1, positions=f(n)), lambda f: cache.plan(n, 3, 1, tables=f(n[:, None])), lambda f: cache.plan(n[:2], 3, 1, starts=f(n)),
             lambda f: cache.truncate(f(n)), lambda f: cache.truncate(n, rows=f(n)), lambda f: cache.append(0, f(x), x), lambda f: cache.append(0, x, f(x)),
             lambda f: cache.attention(0, f(x), out=x), lambda f: cache.attention(0, x, out=f(x)),
             lambda f: cache.attention(0, x, out=x, lse=f(torch.zeros((3, 2)))), lambda f: cache.read_pages(0, f(n), pages), lambda f: cache.read_pages(0, n, f(pages)),
             lambda f: cache.read_pages(0, n, pages, f(pages))]
    for call in calls:
        made = len(cache._L.calls)
        with pytest.raises(ValueError, match="cuda:1"):
            call(there)
        assert len(cache._L.calls) == made
        call(here)
        assert len(cache._L.calls) == made + 1
