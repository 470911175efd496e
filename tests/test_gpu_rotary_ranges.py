"""Rotation at far angles.  Tolerances: tests/test_gpu_rotary.py."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

from qwenquest_amd import QKNormRotary

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
