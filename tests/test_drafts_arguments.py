"""What a drafted step's Python calls hand on: sizes that fit, in front of the C interface, which takes 32 bits of any."""
import math

import pytest

import turboquant_mlx_core_b200 as tq
from tests.test_paged_arguments import cache  # noqa: F401

torch = pytest.importorskip("torch")


class Sized:
    """A contiguous tensor of any size, without memory."""
    is_cuda = True

    def __init__(self, *shape, dtype=torch.int32):
        self.shape, self.dtype = torch.Size(shape), dtype

    def get_device(self):
        return -1

    def data_ptr(self):
        return 4096

    def numel(self):
        return math.prod(self.shape)

    def is_contiguous(self):
        return True

    def stride(self):
        return tuple(math.prod(self.shape[i + 1:]) for i in range(len(self.shape)))


@pytest.mark.parametrize("wide", [1 << 31, 1 << 32, (1 << 32) + 3])
def test_sizes_that_do_not_fit(cache, monkeypatch, wide):  # noqa: F811
    from turboquant_mlx_core_b200 import paged
    monkeypatch.setattr(paged._lib, "load", lambda: cache._L)
    half, f32 = dict(dtype=torch.float16), dict(dtype=torch.float32)
    three = Sized(3)

    def verify(**change):
        rows = change.pop("rows", 3)
        return tq.verify_drafts(**{**dict(starts=Sized(3), parents=Sized(rows), tokens=Sized(rows), target=Sized(rows, 5, **f32), draft=None, uniforms=Sized(rows, **f32),
                                          path=Sized(2, 2), kept=Sized(2), next=Sized(2)), **change})

    def rope(tokens=3, heads=2, dim=64):
        x = Sized(tokens, heads, dim, **half)
        return tq.qk_norm_rope(x, x, Sized(dim, **half), Sized(dim, **half), Sized(tokens))

    calls = [lambda: cache.tree(Sized(wide)), lambda: cache.tree(positions=Sized(wide)), lambda: cache.keep(Sized(wide, 2), Sized(wide)), lambda: cache.keep(Sized(3, wide), three),
             lambda: verify(rows=wide), lambda: verify(path=Sized(2, wide)), lambda: verify(target=Sized(3, wide, **f32)),
             lambda: verify(path=Sized(wide, 2), kept=Sized(wide), next=Sized(wide), starts=Sized(wide + 1)), lambda: rope(tokens=wide), lambda: rope(heads=wide), lambda: rope(dim=wide),
             lambda: cache.tree_attention(0, Sized(wide, 2, 64, **half), out=Sized(wide, 2, 64, **half)), lambda: cache.append(0, Sized(wide, 2, 64, **half), Sized(wide, 2, 64, **half))]
    for call in calls:
        with pytest.raises(ValueError, match="32 bits"):
            call()
    assert cache._L.calls == []
    cache.tree(three)
    cache.keep(Sized(3, 2), three)
    verify()
    rope()
    cache.tree_attention(0, Sized(3, 2, 64, **half), out=Sized(3, 2, 64, **half))
    assert [c[0] for c in cache._L.calls] == ["tq_paged_tree", "tq_paged_keep", "tq_verify_drafts", "tq_qk_norm_rope_f16", "tq_paged_tree_attention"]


@pytest.mark.parametrize("name", ["attention", "tree_attention"])
def test_errors_name_their_call(cache, monkeypatch, name):  # noqa: F811
    monkeypatch.setattr(cache._L, f"tq_paged_{name}", lambda *a: -1, raising=False)
    x = Sized(3, 2, 64, dtype=torch.float16)
    with pytest.raises(tq.TQError, match=rf"PagedKVCache\.{name}\b"):
        getattr(cache, name)(0, x, out=x)
    with pytest.raises(TypeError, match=rf"^{name}: queries"):
        getattr(cache, name)(0, Sized(3, 2, 64, dtype=torch.float32))
