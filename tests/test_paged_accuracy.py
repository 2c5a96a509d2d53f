"""How far the paged cache's numbers are from what was written: what its header says, of the definitions that the kernels equal bit for bit."""
import numpy as np
import pytest

from tests.paged_model import Model


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("uneven", [False, True])
def test_numbers_are_half_a_scale_off_at_most(page, dim, uneven):
    rng = np.random.default_rng(page + dim)
    tokens = 8 * page
    x = rng.standard_normal((tokens, 1, dim))
    if uneven:
        x *= np.exp(0.5 * rng.standard_normal((tokens, 1, 1))) * np.exp(0.4 * rng.standard_normal((1, 1, dim)))
    m = Model(1, dim, 8, page)
    m.plan([tokens])
    m.append(0, x)
    off = np.abs(m.held(0, 0) - x).reshape(8, -1)
    top = np.abs(x).reshape(8, -1).max(1)
    half = np.array([2.0 ** (m.exps[0][p, 0] - 1) for p in m.tables[0]])
    assert (off <= half[:, None]).all() and (half <= top / 127.5).all() and (half > top / 255).all()
    # a rounding to a step of s is s / sqrt(12) off in the mean: between the two ends for the largest magnitudes
    error, norm = np.sqrt((off ** 2).sum()), np.linalg.norm(x)
    assert 0.9 < error / np.sqrt(((2 * half) ** 2 / 12).sum() * page * dim) < 1.1 and error / norm < (0.06 if uneven else 0.02)


def test_a_draft_that_is_taken_back_leaves_its_scale():
    m = Model(1, 64, 2, 16)
    x = np.full((5, 1, 64), 0.3)
    m.plan([5])
    m.append(0, x)
    m.plan([1])
    m.append(0, np.full((1, 1, 64), 127 * 0.5))
    m.truncate([5])
    assert (m.held(0, 0) == 0.5).all()
    m.plan([1])
    m.append(0, x[:1])
    assert (m.held(0, 0) == 0.5).all()
