"""What stands between a layer's QKV product and its attention: RMS norms of each query and key head
and the rotation by position, in one launch (``qq_qk_norm_rotary``).

``AttentionBackend.forward_qkv`` calls it for layers that carry one.
"""

from __future__ import annotations

import math
from collections.abc import Sequence
from fractions import Fraction

import torch
from torch.autograd import forward_ad

from qwenquest_amd import _lib
from qwenquest_amd.paged import _indexed

__all__ = ["QKNormRotary"]

#: quarter turns of a radian, 2 / pi, by 2^160
_QUARTERS = round(2**161 / Fraction("3.14159265358979323846264338327950288419716939937510582097494459"))
_ORDERS = ("blocks", "cycled")
_PAIRS = ("halves", "neighbours")


class QKNormRotary:
    """Norms and rotation of one layer's queries and keys.

    A head x becomes ``y = x / sqrt(mean(x^2) + eps) * weight`` (``q_weight`` / ``k_weight [head_dim]``, copied;
    None: no norm), then of the first ``rotary_dim`` channels pair j turns by ``position * inv_freq[j]``:
    ``(a, b) -> (a cos - b sin, b cos + a sin)``.  In float32, rounded once to the input's type (bfloat16 or float32); an angle
    is off by 2^-53 of itself at most, so that sine and cosine are good to float32's last places up to 2^29 radians
    and to 2^-22 at 2^31.  A token at a position of 2^31 or beyond, either way, gets NaN where it would turn.

    ``inv_freq [rotary_dim / 2]``: by default ``base ** (-2 j / rotary_dim)``.  ``pairs``: "halves" (channel j with
    j + rotary_dim / 2) or "neighbours" (2 j with 2 j + 1).  ``sections``: the number of pairs that turn by each of several
    position axes (time, height, width), in ``section_order`` "blocks" (the first axis's pairs, then the second's) or
    "cycled" (dealt to the axes in turn, as long as each has pairs left).
    """

    def __init__(
        self,
        num_heads: int,
        kv_heads: int,
        head_dim: int,
        *,
        q_weight: torch.Tensor | None = None,
        k_weight: torch.Tensor | None = None,
        eps: float = 1e-6,
        base: float = 10000.0,
        rotary_dim: int | None = None,
        inv_freq: Sequence[float] | torch.Tensor | None = None,
        sections: Sequence[int] | None = None,
        section_order: str = "blocks",
        pairs: str = "halves",
        device: torch.device | str,
    ):
        self.device = _indexed(device)
        if self.device.type != "cuda":
            raise RuntimeError("qwenquest_amd.QKNormRotary needs a GPU device (no CPU path)")
        if not 0 < num_heads < 1 << 16 or not 0 < kv_heads < 1 << 16:
            raise ValueError(f"num_heads and kv_heads must be 1 .. 65535, got {num_heads} and {kv_heads}")
        if head_dim % 8 or not 8 <= head_dim <= 512:
            raise ValueError(f"head_dim must be a multiple of 8 up to 512, got {head_dim}")
        if pairs not in _PAIRS or section_order not in _ORDERS:
            raise ValueError(f"pairs must be one of {_PAIRS} and section_order of {_ORDERS}, got {pairs!r} and {section_order!r}")
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        step = 8 if pairs == "neighbours" else 16
        if not 0 <= rotary_dim <= head_dim or rotary_dim % step:
            raise ValueError(f"rotary_dim must be a multiple of {step} up to head_dim for pairs={pairs!r}, got {rotary_dim}")
        if not 0.0 <= eps < math.inf:
            raise ValueError(f"eps must be finite and not negative, got {eps}")
        count = rotary_dim // 2
        if inv_freq is None:
            if not 0.0 < base < math.inf:
                raise ValueError(f"base must be positive, got {base}")
            freq = torch.tensor([float(base) ** (-2.0 * j / rotary_dim) for j in range(count)], dtype=torch.float64)
        else:
            freq = torch.as_tensor(inv_freq, dtype=torch.float64, device="cpu").flatten()
            if freq.numel() != count or not bool(torch.isfinite(freq).all()):
                raise ValueError(f"inv_freq must hold {count} finite frequencies, one for each pair")
        left = [count] if sections is None else [int(s) for s in sections]
        if not left or min(left) < 0 or sum(left) != count:
            raise ValueError(f"sections {tuple(left)} must add up to the {count} pairs")
        self.num_heads, self.kv_heads, self.head_dim, self.rotary_dim = num_heads, kv_heads, head_dim, rotary_dim
        self.eps, self.axes, self.neighbours = float(eps), len(left), pairs == "neighbours"
        # in quarter turns, as the kernel takes angles
        self._quarters = torch.tensor([_quarter_turns(f) for f in freq.tolist()], dtype=torch.float64).to(self.device)
        self._axis = torch.tensor(_deal(left, section_order == "cycled"), dtype=torch.int32, device=self.device)
        self._weights = [self._weight(w, what) for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight"))]
        self._bind()

    def _bind(self) -> None:
        """What every call passes, of tensors that stay where they are."""
        self._args = (*(_lib.ptr(w) for w in self._weights), self.eps, _lib.ptr(self._quarters), _lib.ptr(self._axis),
                      self.rotary_dim // 2, int(self.neighbours))

    def __getstate__(self) -> dict:  # addresses hold for this object's own tensors, not for a copy's or a pickle's
        return {name: value for name, value in self.__dict__.items() if name != "_args"}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._bind()

    def _weight(self, w: torch.Tensor | None, what: str) -> torch.Tensor | None:
        if w is None:
            return None
        if w.shape != (self.head_dim,) or not w.dtype.is_floating_point:
            raise ValueError(f"{what} must hold {self.head_dim} floating-point values, got {tuple(w.shape)} {w.dtype}")
        return w.detach().to(device=self.device, dtype=torch.float32, copy=True).contiguous()

    def __call__(self, qkv: torch.Tensor, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """``qkv [n, (num_heads + 2 kv_heads) * head_dim]``, a token's query heads, key heads and value heads in a
        row, at ``positions`` (``[n]``, or ``[axes, n]``) -> ``q [n, num_heads, head_dim]``, ``k`` and ``v [n, kv_heads,
        head_dim]``, dense (v as it was)."""
        _lib.refuse_tracing("QKNormRotary")
        h, kv, dim = self.num_heads, self.kv_heads, self.head_dim
        if qkv.dim() != 2 or qkv.shape[1] != (h + 2 * kv) * dim:
            raise ValueError(f"qkv must be [n, ({h} + 2 * {kv}) * {dim}], got {tuple(qkv.shape)}")
        qkv, ptr, stride, size = self._rows(qkv)
        n, step = qkv.shape[0], dim * size
        return self._launch((ptr, stride, ptr + h * step, stride, ptr + (h + kv) * step, stride), qkv.dtype, n, positions, 3)

    def apply(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """``q [n, num_heads, head_dim]`` and ``k [n, kv_heads, head_dim]`` (or with the heads in a row) at
        ``positions``, as new dense tensors."""
        _lib.refuse_tracing("QKNormRotary")
        rows, args = [], []
        for x, heads, what in ((q, self.num_heads, "q"), (k, self.kv_heads, "k")):
            if x.dim() == 3 and x.shape[1:] == (heads, self.head_dim):
                # a view wherever a token's heads lie in a row
                x = x.reshape(x.shape[0], heads * self.head_dim)
            if x.dim() != 2 or x.shape[1] != heads * self.head_dim:
                raise ValueError(f"{what} must be [n, {heads}, {self.head_dim}], got {tuple(x.shape)}")
            x, ptr, stride, _ = self._rows(x)
            rows.append(x)
            args += [ptr, stride]
        if rows[0].shape[0] != rows[1].shape[0] or rows[0].dtype != rows[1].dtype:
            raise ValueError("q and k differ in tokens or type")
        return self._launch((*args, None, 0), rows[0].dtype, rows[0].shape[0], positions, 2)

    def _rows(self, x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
        """``x [n, width]`` with rows that the kernel takes: itself or a copy; its address, row stride and element size."""
        if x.device != self.device:
            raise ValueError(f"the heads lie on {x.device}, the weights and frequencies on {self.device}")
        if (x.requires_grad and torch.is_grad_enabled()) or forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError("QKNormRotary computes no gradients: detach its inputs or call it under torch.no_grad()")
        size, (n, width), (stride, unit) = x.element_size(), x.shape, x.stride()
        if n <= 1:
            stride = width
        if unit != 1 or x.data_ptr() % 16 or stride * size % 16 or stride < 0:
            x, stride = x.clone(memory_format=torch.contiguous_format), width
        return x, x.data_ptr(), stride, size

    def _launch(self, rows: tuple, dtype: torch.dtype, n: int, pos: torch.Tensor, outputs: int) -> tuple[torch.Tensor, ...]:
        dev, code = self.device, _lib.dtype_code(dtype)
        if pos.dtype.is_floating_point or pos.dtype == torch.bool:
            raise ValueError(f"positions must hold whole numbers, got {pos.dtype}")
        if pos.shape != ((n,) if self.axes == 1 and pos.dim() == 1 else (self.axes, n)):
            raise ValueError(f"positions must be [{self.axes}, {n}]{f' or [{n}]' if self.axes == 1 else ''}, got {tuple(pos.shape)}")
        if pos.dtype != torch.int64 or pos.device != dev or not pos.is_contiguous():
            pos = pos.to(device=dev, dtype=torch.int64).contiguous()
        outs = tuple(torch.empty((n, heads, self.head_dim), dtype=dtype, device=dev)
                     for heads in (self.num_heads, self.kv_heads, self.kv_heads)[:outputs])
        with _lib.on(dev):
            _lib.call("qq_qk_norm_rotary", *rows, code, self.num_heads, self.kv_heads, self.head_dim, n, *self._args,
                      pos.data_ptr(), n, self.axes, *(o.data_ptr() for o in outs), *([None] * (3 - outputs)), _lib.stream(dev))
        return outs


def _quarter_turns(radians: float) -> float:
    """``radians`` in quarter turns, by a product of whole numbers: rounded once."""
    mantissa, exponent = math.frexp(radians)
    return math.ldexp(float(int(mantissa * 2**53) * _QUARTERS), exponent - 53 - 160)


def _deal(left: list[int], cycled: bool) -> list[int]:
    """The axis of each pair."""
    if not cycled:
        return [axis for axis, count in enumerate(left) for _ in range(count)]
    left, out, axis = list(left), [], 0
    while sum(left):
        if left[axis]:
            out.append(axis)
            left[axis] -= 1
        axis = (axis + 1) % len(left)
    return out
