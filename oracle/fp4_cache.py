"""The 4-bit block cache by its definition, in float64 numpy.

Blocks of 64 tokens; of a token and KV head K has for each 32 channels, V as a whole an exponent e, the least
with max |x| <= 7 * 2^e within K's -96 .. 125 or V's -50 .. 59, and values that are the nearest of
+-{0, 1/2, 1, 3/2, 2, 3, 4, 6} * 2^e, ties to the even code, 6 * 2^e beyond it.  A token and head whose K or V
is not finite, or whose V is above 7 * 2^59, is lost: NaN in K and in V.
"""

from __future__ import annotations

import numpy as np

BLOCK = 64
GROUP = 32
K_EXP, V_EXP = (-96, 125), (-50, 59)
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def exponent(amax: np.ndarray, span: tuple[int, int]) -> np.ndarray:
    """Least e with amax <= 7 * 2^e, within span."""
    mant, e = np.frexp(np.asarray(amax, dtype=np.float64) / 7.0)  # amax / 7 = mant * 2^e, mant in [1/2, 1)
    e = np.where(mant == 0.5, e - 1, e)
    return np.where(np.asarray(amax) == 0.0, span[0], np.clip(e, *span)).astype(np.int64)


def round_e2m1(y: np.ndarray) -> np.ndarray:
    """The nearest e2m1 value, ties to the even code, 6 beyond it."""
    a = np.abs(y)
    code = np.zeros(a.shape, dtype=np.int64)
    for i in range(7):
        border = (GRID[i] + GRID[i + 1]) / 2
        code += (a > border) | ((a == border) & (i % 2 == 1))
    return np.copysign(GRID[code], y)


def quantise(x: np.ndarray, group: int, span: tuple[int, int]) -> np.ndarray:
    """``x [..., D]`` as the cache keeps it, one exponent for ``group`` channels."""
    y = x.astype(np.float64).reshape(*x.shape[:-1], -1, group)
    e = exponent(np.abs(y).max(-1, keepdims=True), span)
    return np.ldexp(round_e2m1(np.ldexp(y, -e)), e).reshape(x.shape)


class Cache:
    """One layer: values [blocks, 64, KV, D] of K and V."""

    def __init__(self, blocks: int, kv: int, dim: int):
        self.blocks = blocks
        self.values = [np.zeros((blocks, BLOCK, kv, dim)) for _ in range(2)]

    def write(self, loc, k: np.ndarray, v: np.ndarray) -> None:
        with np.errstate(invalid="ignore"):
            good = np.isfinite(k).all(-1) & (np.abs(v) <= 7 * 2.0 ** V_EXP[1]).all(-1)
        for which, (x, group, span) in enumerate(((k, GROUP, K_EXP), (v, v.shape[-1], V_EXP))):
            x = quantise(np.where(good[..., None], x, 0.0), group, span)
            x[~good] = np.nan
            for i, row in enumerate(np.asarray(loc, dtype=np.int64)):  # the last entry of a row counts
                if 0 < row // BLOCK < self.blocks:
                    self.values[which][row // BLOCK, row % BLOCK] = x[i]

    def rows(self, loc) -> tuple[np.ndarray, np.ndarray]:
        loc = np.asarray(loc, dtype=np.int64)
        return tuple(x[loc // BLOCK, loc % BLOCK].copy() for x in self.values)
