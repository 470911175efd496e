"""The 8-bit block cache and its operators by their definitions, in float64 numpy.

Blocks of 64 tokens; per (block, KV head), K and V apart, e4m3 codes and a scale 2^e.  A write puts
values x into a block: e becomes the largest of the exponent before (-110 where the write holds the
block's first row, which begins the block) and the least e >= -110 with max |x| <= 448 * 2^e; the
block's other values are rounded again when e grows.  Values that are not finite make the scale NaN
until the block is begun again.
"""

from __future__ import annotations

import numpy as np

BLOCK = 64
E_MIN = -110
TOP = 448.0


def exponent(amax: float) -> int:
    """Least e >= E_MIN with amax <= 448 * 2^e."""
    if amax == 0.0:
        return E_MIN
    mant, e = np.frexp(amax / TOP)  # amax / 448 = mant * 2^e, mant in [1/2, 1)
    return max(int(e) - (1 if mant == 0.5 else 0), E_MIN)


def round_e4m3(y: np.ndarray) -> np.ndarray:
    """|y| <= 448 to the nearest e4m3 value, ties to even: 4 significand bits, steps of 2^-9 at least."""
    _, e = np.frexp(y)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.round(y / step) * step


class Cache:
    """One layer: values [blocks, 64, KV, D] and exponents [blocks, KV] of K and V, NaN flags."""

    def __init__(self, blocks: int, kv: int, dim: int):
        self.blocks = blocks
        self.values = [np.zeros((blocks, BLOCK, kv, dim)) for _ in range(2)]
        self.expo = [np.full((blocks, kv), E_MIN) for _ in range(2)]
        self.lost = [np.zeros((blocks, kv), dtype=bool) for _ in range(2)]

    def scale(self, which: int) -> np.ndarray:
        return np.where(self.lost[which], np.nan, np.ldexp(1.0, self.expo[which]))

    def write(self, loc, k: np.ndarray, v: np.ndarray) -> None:
        loc = np.asarray(loc, dtype=np.int64)
        i = 0
        while i < len(loc):
            j = i
            while j < len(loc) and loc[j] // BLOCK == loc[i] // BLOCK:
                j += 1
            block = int(loc[i] // BLOCK)
            if 0 < block < self.blocks:
                slots: dict[int, int] = {int(loc[t] % BLOCK): t for t in range(i, j)}  # the last entry counts
                for which, x in enumerate((k, v)):
                    self._write_block(which, block, list(slots), x[list(slots.values())].astype(np.float64))
            i = j

    def _write_block(self, which: int, block: int, slots: list[int], x: np.ndarray) -> None:
        values, expo, lost = self.values[which][block], self.expo[which][block], self.lost[which][block]
        begun = 0 in slots
        for h in range(x.shape[1]):
            xh = x[:, h]
            ok = np.isfinite(xh)
            if begun:
                values[:, h], expo[h], lost[h] = 0.0, E_MIN, False
            e = max(int(expo[h]), exponent(float(np.abs(np.where(ok, xh, 0.0)).max())))
            if e > expo[h]:
                values[:, h] = np.ldexp(round_e4m3(np.ldexp(values[:, h], -e)), e)
            expo[h] = e
            lost[h] |= not ok.all()
            values[slots, h] = np.ldexp(round_e4m3(np.ldexp(np.where(ok, xh, 0.0), -e)), e)

    def rows(self, loc) -> tuple[np.ndarray, np.ndarray]:
        loc = np.asarray(loc, dtype=np.int64)
        out = []
        for which in range(2):
            x = self.values[which][loc // BLOCK, loc % BLOCK].copy()
            x[self.lost[which][loc // BLOCK]] = np.nan
            out.append(x)
        return out[0], out[1]


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float):
    """``q [H, D]`` over ``k, v [n, KV, D]`` in float64.  Returns out [H, D], and for the error bounds
    sum p |v| / sum p [H, D] and the largest sum |q k| |scale| over the rows [H]."""
    H, D = q.shape
    n, kv, _ = k.shape
    out, spread, size = np.zeros((H, D)), np.zeros((H, D)), np.zeros(H)
    if n == 0:
        return out, spread, size
    q = q.astype(np.float64)
    for h in range(H):
        kh, vh = k[:, h // (H // kv)], v[:, h // (H // kv)]
        s = kh @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], spread[h] = p @ vh, p @ np.abs(vh)
        size[h] = (np.abs(kh) @ np.abs(q[h])).max() * abs(scale)
    return out, spread, size


def attend_tolerance(out, spread, size, n: int, dim: int, bf16_out: bool, weight_bits: int) -> np.ndarray:
    """How far a kernel may be off ``attend``, by its roundings: half a step of the output; the weights
    to ``weight_bits`` significand bits by truncation (off by 2^-(weight_bits - 2) of a weight at
    most, in pieces); scores as float32 sums of dim products, each partial sum half a step off
    (numerator and denominator both move by the score's error); float32 sums of n weights, by 64
    lanes first."""
    half = 2.0**-8 if bf16_out else 2.0**-24
    score = (dim + 4) * 2.0**-23 * size
    rel = 2.0 ** -(weight_bits - 2) + (n / 64 + 64) * 2.0**-23 + 2 * score
    return half * np.abs(out) + rel[:, None] * spread + 1e-38


class Slots:
    """The paged request pool on the host: block lists, a stack of free blocks."""

    def __init__(self, reqs: int, width: int, num_blocks: int):
        self.width = width
        self.stack = list(range(num_blocks - 1, 0, -1))
        self.memory = list(self.stack)  # the stack's memory keeps what was taken off it
        self.table = [[] for _ in range(reqs)]
        self.r2t = np.zeros((reqs, width), dtype=np.int64)

    def _refused(self, reqs, ends) -> bool:
        named = [r for r, e in zip(reqs, ends) if e is not None]
        if len(set(named)) < len(named) or any(r < 0 or r >= len(self.table) for r in named):
            return True
        if any(e is not None and (e[0] < 0 or e[1] < e[0] or e[1] > self.width) for e in ends):
            return True
        need = sum(max(0, -(-e[1] // BLOCK) - len(self.table[r])) for r, e in zip(reqs, ends) if e is not None)
        return need > len(self.stack)

    def assign(self, reqs, prefix, new, total: int):
        ends = [None if n == 0 else (p, p + n) for p, n in zip(prefix, new)]
        loc, pos = np.zeros(total, dtype=np.int64), np.zeros(total, dtype=np.int64)
        if self._refused(reqs, ends) or sum(new) > total:
            return loc, pos
        at = 0
        for r, e in zip(reqs, ends):
            if e is None:
                continue
            while len(self.table[r]) * BLOCK < e[1]:
                self.table[r].append(self.stack.pop())
            for p in range(*e):
                loc[at] = self.table[r][p // BLOCK] * BLOCK + p % BLOCK
                pos[at] = p
                self.r2t[r, p] = loc[at]
                at += 1
        return loc, pos

    def release(self, reqs) -> None:
        if len(set(reqs)) < len(reqs) or any(r < 0 or r >= len(self.table) for r in reqs):
            return
        back = [b for r in reqs for b in self.table[r]]
        for r in reqs:
            self.r2t[r, : len(self.table[r]) * BLOCK] = 0
            self.table[r] = []
        self.stack += back[::-1]
        self.memory[: len(self.stack)] = self.stack
