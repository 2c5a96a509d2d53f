"""GPU tests of the norms' rotation at positions up to 2^31, against angles in 60 digits."""
from decimal import Decimal, getcontext

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def pi():
    """Machin: 16 atan(1/5) - 4 atan(1/239)."""
    def atan(n):
        x, total, k, term = Decimal(1) / n, Decimal(0), 0, Decimal(1) / n
        while abs(term) > Decimal(10) ** -70:
            total += term / (2 * k + 1)
            term, k = -term * x * x, k + 1
        return total
    return 16 * atan(5) - 4 * atan(239)


def angles(positions, theta, dim):
    """[positions, dim / 2] in radians, within a turn."""
    getcontext().prec = 70
    turn, log = 2 * pi(), Decimal(theta).ln()
    out = np.zeros((len(positions), dim // 2))
    for i in range(dim // 2):
        frequency = (log * -2 * i / dim).exp() / turn
        for r, p in enumerate(positions):
            fraction = Decimal(int(p)) * frequency
            out[r, i] = float((fraction - fraction.to_integral_value()) * turn)
    return out


@pytest.mark.parametrize("theta,dim", [(10.0, 64), (1e4, 128), (1e6, 80), (5e8, 128), (5e8, 512)])
def test_positions_up_to_the_largest(tq, theta, dim):
    """Frequencies are computed in 64-bit floats: a power that is a unit of 2^-52 off at most, a division by 2 pi and its rounding, and up to seven
    products with a ratio that is a unit off, 25 2^-53 of a frequency in all, of 1 / (2 pi) turns at most: below 2^-51 turns times the position,
    beside the roundings that the docstring of
    drafts_model.qk_norm_rope counts."""
    rng = np.random.default_rng(dim)
    positions = [0, 1, -1, 1 << 24, (1 << 24) + 1, 1 << 28, -(1 << 30) + 7, (1 << 31) - 1, -(1 << 31), 2000000011, 987654321]
    x = [rng.standard_normal((len(positions), h, dim)).astype(np.float16) for h in (3, 1)]
    w = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float16) for _ in range(2)]
    got = tq.qk_norm_rope(*(torch.from_numpy(t).cuda() for t in (*x, *w)), torch.tensor(positions, dtype=torch.int32, device="cuda"), theta=theta, eps=1e-6)
    angle = angles(positions, theta, dim)[:, None]
    far = (np.abs(np.asarray(positions, np.float64)) * 2.0 ** -51 * 2 * np.pi)[:, None, None]
    for g, t, v in zip(got, x, w):
        t, v = t.astype(np.float64), v.astype(np.float64)
        y = t / np.sqrt((t ** 2).mean(2, keepdims=True) + 1e-6) * v
        a, b = y[..., :dim // 2], y[..., dim // 2:]
        want = np.concatenate([a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)], 2)
        size = np.concatenate([np.abs(a) + np.abs(b)] * 2, 2)
        off = size * (dim / 2 + 17) * 2.0 ** -24 + size * far
        tol = (np.abs(want) + off) * 2.0 ** -11 + 2.0 ** -25 + off
        worst = np.max(np.abs(g.cpu().numpy().astype(np.float64) - want) / tol)
        assert worst <= 1, f"off by {worst} times the bound"
