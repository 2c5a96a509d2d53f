"""The definitions of a drafted decoding step, and what of its calls is refused before any device work."""
import numpy as np
import pytest

import turboquant_mlx_core_b200 as tq
from tests import drafts_model
from tests.paged_model import Model
from tests.test_paged_arguments import cache  # noqa: F401
from tests.test_paged_devices import Elsewhere

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("drawn", [True, False])
def test_tokens_are_distributed_as_the_target_has_them(drawn):
    """The first token behind node 0 (an accepted child's, or the one that follows) and, behind an accepted child, the next one: each is
    within five standard deviations of its share (of 12 numbers, once in 150 thousand runs it is not)."""
    rng = np.random.default_rng(5)
    p, q = rng.dirichlet(np.ones(6)), rng.dirichlet(np.ones(6))
    rows_p, rows_q, n = np.stack([p, rng.dirichlet(np.ones(6)), p[::-1], p]), np.stack([q] * 4), 20000
    first, second, went = np.zeros(6), np.zeros(6), 0
    for _ in range(n):
        x = rng.choice(6, 3, p=q) if drawn else [1, 4, 2]
        tokens = [0, *x]
        path, nxt = drafts_model.verify([-1, 0, 0, 0], tokens, rows_p, rows_q if drawn else None, rng.random(4), 4)
        first[tokens[path[1]] if len(path) > 1 else nxt] += 1
        if len(path) > 1 and path[1] == 1:
            second[nxt] += 1
            went += 1
    for got, share, total in ((first, p, n), (second, rows_p[1], went)):
        assert (np.abs(got - total * share) < 5 * np.sqrt(total * share * (1 - share))).all() and total > 100


def test_kept_tokens_keep_their_values_within_a_page_and_join_another_one():
    m = Model(1, 64, 4, 16)
    m.plan([14])
    x = np.full((14, 1, 64), 1.0)
    m.append(0, x)
    m.plan([8])
    new = np.arange(1, 9)[:, None, None] * np.ones((8, 1, 64))
    m.append(0, new)
    assert m.exps[0][m.tables[0][0], 0] == -5 and m.exps[0][m.tables[0][1], 0] == -3      # 2 / 2^-5 = 64, 8 / 2^-3 = 64
    drafts_model.keep(m, 0, [[1, 4, 7]])
    m.truncate(drafts_model.kept_lengths(m, [[1, 4, 7]]))
    assert m.lengths[0] == 17 and m.exps[0][m.tables[0][0], 0] == -4
    assert m.held(0, 0)[:, 0, 0].tolist() == [1.0] * 14 + [2.0, 5.0, 8.0]


def test_ancestors_and_depths():
    par = [-1, 0, 0, 1, 3, 2, -1, 6]
    assert drafts_model.depths(par) == [0, 1, 1, 2, 3, 2, 0, 1]
    assert drafts_model.ancestors(par)[4].tolist() == [True, True, False, True, True, False, False, False]


def test_null_and_impossible_arguments():
    L = tq.load()
    one = np.ones(4, np.int32)
    at = one.ctypes.data
    for rc in (L.tq_paged_tree(None, None, 1, None, None), L.tq_paged_keep(None, None, 1, None, 1, None, None)):
        assert rc != 0 and b"NULL" in L.tq_last_error()
    rope = lambda rows=1, qh=2, kh=1, dim=64, qs=128, ks=64, eps=1e-6, theta=1e4, qt=128, kt=64: L.tq_qk_norm_rope_f16(      # noqa: E731
        at, at, at, at, at, rows, qh, kh, dim, qs, ks, eps, theta, at, at, qt, kt, None)
    for change, what in (({"rows": -1}, b"rows"), ({"rows": 1 << 31}, b"rows"), ({"qh": 0}, b"heads"), ({"kh": -1}, b"heads"), ({"kh": 65537}, b"heads"),
                         ({"dim": 40}, b"head_dim"), ({"dim": 0}, b"head_dim"), ({"dim": 528}, b"head_dim"), ({"qs": 127}, b"stride"), ({"ks": 63}, b"stride"),
                         ({"qt": 127}, b"stride"), ({"kt": 63}, b"stride"), ({"eps": -1e-6}, b"eps"), ({"eps": float("nan")}, b"eps"), ({"theta": 1.0}, b"theta"),
                         ({"theta": float("inf")}, b"theta"), ({}, b"device pointers")):
        assert rope(**change) != 0 and what in L.tq_last_error()
    assert rope(rows=0) == 0
    verify = lambda n=1, rows=1, dtype=0, vocab=4, ts=4, ds=4, width=1, draft=at: L.tq_verify_drafts(      # noqa: E731
        at, at, at, n, rows, at, draft, dtype, vocab, ts, ds, at, at, width, at, at, None)
    for change, what in (({"n": -1}, b"requests"), ({"n": 65537}, b"requests"), ({"rows": -1}, b"rows"), ({"vocab": 0}, b"vocabulary"),
                         ({"vocab": (1 << 20) + 1, "ts": 1 << 21, "ds": 1 << 21}, b"vocabulary"), ({"width": 0}, b"path"), ({"dtype": 7}, b"fp32"), ({"ts": 3}, b"stride"),
                         ({"ds": 3}, b"stride"), ({}, b"device pointers")):
        assert verify(**change) != 0 and what in L.tq_last_error(), change
    assert verify(n=0) == 0


def test_python_arguments(cache):  # noqa: F811
    ints = torch.zeros(3, dtype=torch.int32)
    path = torch.zeros((3, 2), dtype=torch.int32)
    cache.tree(ints, positions=ints)
    cache.keep(path, ints, lengths=ints)
    assert [c[0] for c in cache._L.calls] == ["tq_paged_tree", "tq_paged_keep"] and cache._L.calls[0][1][2] == 3 and cache._L.calls[1][1][2] == 2
    for call in (lambda: cache.tree(ints.long()), lambda: cache.keep(path.long(), ints), lambda: cache.keep(path, ints.long())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: cache.tree(path), lambda: cache.tree(ints, positions=ints[:2]), lambda: cache.keep(ints, ints), lambda: cache.keep(path, ints[:2]),
                 lambda: cache.keep(path.T, ints[:2]), lambda: cache.keep(path, ints, lengths=ints[:1]), lambda: cache.tree(torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            call()
    cache._device = 0
    here, there = (lambda t: Elsewhere(t, 0)), Elsewhere
    for call in (lambda f: cache.tree(f(ints)), lambda f: cache.tree(here(ints), positions=f(ints)), lambda f: cache.keep(f(path), here(ints)),
                 lambda f: cache.keep(here(path), f(ints)), lambda f: cache.keep(here(path), here(ints), lengths=f(ints))):
        with pytest.raises(ValueError, match="cuda:1"):
            call(there)
        call(here)


def test_python_arguments_of_functions():
    half, ints = dict(dtype=torch.float16), dict(dtype=torch.int32)
    q, k, w, pos = torch.zeros((3, 4, 64), **half), torch.zeros((3, 2, 64), **half), torch.zeros(64, **half), torch.zeros(3, **ints)
    for args, error in (((q.float(), k, w, w, pos), TypeError), ((q, k.float(), w, w, pos), TypeError), ((q, k, w.float(), w, pos), TypeError),
                        ((q, k, w, w, pos.long()), TypeError), ((q[:2], k, w, w, pos), ValueError), ((q, k[:, :, :32], w, w, pos), ValueError),
                        ((q, k, w[:32], w, pos), ValueError), ((q, k, w, w, pos[:2]), ValueError), ((q.transpose(0, 1), k, w, w, pos), ValueError),
                        ((q, Elsewhere(k), w, w, pos), ValueError), ((q, k, Elsewhere(w), w, pos), ValueError), ((q, k, w, w, Elsewhere(pos)), ValueError),
                        ((q[0], k, w, w, pos), ValueError), ((q, k, w, w, pos), tq.TQError)):       # (the last: host memory)
        with pytest.raises(error):
            tq.qk_norm_rope(*args)
    with pytest.raises(ValueError):
        tq.qk_norm_rope(q, k, w, w, pos, out=(q[:, :2], k))
    rows = torch.zeros((5, 9))
    good = dict(starts=pos, parents=torch.zeros(5, **ints), tokens=torch.zeros(5, **ints), target=rows, draft=rows, uniforms=torch.zeros(5),
                path=torch.zeros((2, 3), **ints), kept=torch.zeros(2, **ints), next=torch.zeros(2, **ints))
    for change, error in (({"starts": pos[:2]}, ValueError), ({"parents": pos}, ValueError), ({"target": rows.double()}, ValueError), ({"target": rows[:4]}, ValueError),
                          ({"draft": rows.half()}, ValueError), ({"draft": rows[:, :8]}, ValueError), ({"uniforms": torch.zeros(4)}, ValueError),
                          ({"uniforms": torch.zeros(5).half()}, ValueError), ({"path": pos}, ValueError), ({"kept": pos}, ValueError), ({"next": pos.long()[:2]}, TypeError),
                          ({"target": rows.double(), "draft": rows.double()}, TypeError), ({"target": rows.T.contiguous().T}, ValueError),
                          ({"draft": Elsewhere(rows)}, ValueError), ({"kept": Elsewhere(good["kept"])}, ValueError), ({}, tq.TQError)):
        with pytest.raises(error):
            tq.verify_drafts(**{**good, **change})
