"""Per-forward batch carrier (reference ``src/qwenquest/batch.py:27-64``)."""

from __future__ import annotations

import enum
from dataclasses import dataclass
from typing import TYPE_CHECKING, Any, NamedTuple

import torch

from qwenquest_amd import _lib

if TYPE_CHECKING:
    from qwenquest_amd.memory import MHATokenToKVPool, ReqToTokenPool

__all__ = ["DecodePlan", "ForwardBatch", "ForwardMode"]


class ForwardMode(enum.Enum):
    EXTEND = "extend"
    DECODE = "decode"

    def is_extend(self) -> bool:
        return self is ForwardMode.EXTEND

    def is_decode(self) -> bool:
        return self is ForwardMode.DECODE


class DecodePlan(NamedTuple):
    """A decode batch of ``bs`` requests over an 8- or 4-bit pool, divided for the chip once for a step's
    layers.  It holds for the stream that made it, and inside a graph capture for what that same
    capture records: elsewhere its memory may not be written yet, or no longer be its own."""

    bs: int
    workspace: torch.Tensor
    stream: int
    #: the capture's number (``_lib.capture_id``), 0 outside of any
    captured: int
    #: tokens that a longer context selects (Quest), or 0: contexts are whole
    top_k: int = 0

    def usable(self, stream: int) -> bool:
        return self.stream == stream and self.captured == _lib.capture_id(self.workspace.device, stream) >= 0


@dataclass
class ForwardBatch:
    """``seq_lens`` counts the token being decoded (its K/V lands at ``seq_len - 1``)."""

    forward_mode: ForwardMode
    input_ids: torch.Tensor | None
    positions: torch.Tensor | None
    req_pool_indices: torch.Tensor  # [bs] int64
    seq_lens: torch.Tensor  # [bs] int64
    out_cache_loc: torch.Tensor | None
    req_to_token_pool: ReqToTokenPool
    token_to_kv_pool: MHATokenToKVPool
    attn_backend: Any
    extend_prefix_lens: torch.Tensor | None = None
    extend_seq_lens: torch.Tensor | None = None
    #: set by a backend's init_forward_metadata: a decode step's work, divided once for its layers
    decode_plan: DecodePlan | None = None

    @property
    def batch_size(self) -> int:
        return int(self.req_pool_indices.shape[0])

    def extend_token_offsets(self) -> list[int]:
        assert self.extend_seq_lens is not None
        offsets = [0]
        for n in self.extend_seq_lens.tolist():
            offsets.append(offsets[-1] + int(n))
        return offsets
