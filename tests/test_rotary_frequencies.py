"""Frequencies in quarter turns, as the rotation's kernel takes them: the nearest float64, by rational arithmetic."""

from __future__ import annotations

import math
import random
from fractions import Fraction

from qwenquest_amd.rotary import _quarter_turns

PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def test_a_frequency_is_rounded_once():
    rng = random.Random(1)
    freqs = [rng.choice([-1.0, 1.0]) * math.exp(rng.uniform(-600, 600)) for _ in range(3000)]
    freqs += [1e4 ** (-j / 64) for j in range(64)] + [0.0, 1.0, -1.0, math.pi / 2, 1.7e308, 2.0**-1000]
    assert [_quarter_turns(f) for f in freqs] == [float(Fraction(f) * 2 / PI) for f in freqs]
