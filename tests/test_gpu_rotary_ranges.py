"""Head norms and rotation at far angles, and of rows of any size without an epsilon.  Tolerances: tests/test_gpu_rotary.py."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

from qwenquest_amd import QKNormRotary
from tests.test_gpu_rotary import check

pytestmark = pytest.mark.gpu

PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def reduced(pos, freq):
    """pos * freq radians, an exact product, less whole turns: in float64, off by its own rounding alone."""
    out = np.empty((len(pos), len(freq)))
    for j, f in enumerate(freq):
        f = Fraction(float(f))
        for i, p in enumerate(pos):
            t = int(p) * f
            out[i, j] = float(t - 2 * PI * round(t / (2 * PI)))
    return out


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("low, high", [(0.5, 1.0), (1e-3, 1e-2), (1e3, 1e5)])
def test_angles_are_off_by_a_rounding_of_float64_at_most(cuda, low, high, neighbours):
    """Products of up to 31 and 53 bits against rational arithmetic.  A frequency in quarter turns is rounded once, which
    is 2^-53 of the angle; the rest as for near positions: of sine and cosine 2^-22 and of the rotation's three roundings two half steps,
    of the larger of a pair."""
    rng = np.random.default_rng(int(high * 1000))
    freq = np.exp(rng.uniform(np.log(low), np.log(high), 32)) * rng.choice([-1.0, 1.0], 32)
    pos = np.concatenate([rng.integers(-(1 << 31) + 1, 1 << 31, 250), rng.integers((1 << 31) - 1000, 1 << 31, 150),
                          rng.integers(-50, 50, 20), [(1 << 31) - 1, 1 - (1 << 31)]])
    op = QKNormRotary(1, 1, 64, inv_freq=torch.from_numpy(freq), pairs="neighbours" if neighbours else "halves", device=cuda)
    x = torch.randn(len(pos), 3 * 64, device=cuda)
    q, k, _ = op(x, torch.from_numpy(pos).to(cuda))
    t = reduced(pos, freq)
    for got, part in ((q, x[:, :64]), (k, x[:, 64:128])):
        y, got = part.double().cpu().numpy(), got[:, 0].double().cpu().numpy()
        a, b = (y[:, 0::2], y[:, 1::2]) if neighbours else (y[:, :32], y[:, 32:])
        ga, gb = (got[:, 0::2], got[:, 1::2]) if neighbours else (got[:, :32], got[:, 32:])
        size = np.hypot(a, b)
        tol = (2.0**-22 + 2 * 2.0**-24 + 2.0**-53 * np.abs(pos[:, None] * freq)) * size
        for g, want in ((ga, a * np.cos(t) - b * np.sin(t)), (gb, b * np.cos(t) + a * np.sin(t))):
            err = np.abs(g - want) / (tol + 2.0**-24 * np.abs(want))
            assert err.max() <= 1, f"off by {err.max():.2f} tolerances at {np.unravel_index(err.argmax(), err.shape)}"


@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-30, 1e-6, 1e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [8, 80, 128, 512])
def test_rows_of_any_size_are_normed(cuda, dim, dtype, eps):
    """Rows from float32's least numbers to its largest: their squares leave its range either way."""
    least = [2.0**-149, 1e-42] if dtype == torch.float32 else [2.0**-133, 1e-39]
    sizes = [*least, 1e-38, 1e-30, 1e-20, 1e-18, 1e-15, 1.0, 1e10, 1e18, 1e19, 1e25, 1e30, 3e37]
    w = 0.5 + torch.rand(dim, device=cuda)
    op = QKNormRotary(len(sizes), 1, dim, q_weight=w, k_weight=w, eps=eps, rotary_dim=dim // 16 * 16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(dim)
    x = torch.empty((3, len(sizes) + 2, dim), device=cuda, dtype=torch.float64).uniform_(-3.0, 3.0, generator=gen)
    x[..., 1] = 1.0
    x[:, : len(sizes)] *= torch.tensor(sizes, device=cuda, dtype=torch.float64)[:, None]
    x = x.to(dtype)
    assert (x[:, : len(sizes)] != 0).any(-1).all() and x.isfinite().all()
    pos = torch.tensor([0, 5, 1000], device=cuda)
    q, k, _ = op(x.view(3, -1), pos)
    P = op.rotary_dim // 2
    freq = 1e4 ** (-2.0 * np.arange(P) / max(op.rotary_dim, 1))
    at = pos.cpu().numpy()[None]
    eps32 = float(np.float32(eps))  # as the C entry takes it
    for got, part in ((q, x[:, : len(sizes)]), (k, x[:, len(sizes) : -1])):
        check(got, part, w, eps32, freq, [0] * P, at, False)


def test_rows_that_cannot_be_normed(cuda):
    """Without an epsilon a row of zeros has no norm; what is not finite spoils its row alone."""
    op = QKNormRotary(4, 1, 64, q_weight=torch.ones(64), k_weight=torch.ones(64), eps=0.0, device=cuda)
    x = torch.ones(1, 6, 64, device=cuda)
    x[0, 0], x[0, 1, 3], x[0, 2, 3] = 0.0, float("inf"), float("nan")
    q, k, _ = op(x.view(1, -1), torch.tensor([1], device=cuda))
    assert q[0, 0].isnan().all() and q[0, 1, [3, 35]].isnan().all() and q[0, 2].isnan().all()
    assert q[0, 3].isfinite().all() and k.isfinite().all()
