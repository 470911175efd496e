"""Pools whose rows come in blocks of 64 tokens: request tables built on the GPU, and K/V pools
held in 8 or 4 bits.

``BlockReqToTokenPool`` is ``ReqToTokenPool`` with a device allocator: it hands out whole blocks
from the requests' lengths and writes the block table, ``req_to_token`` and the slot map of a
batch's new tokens in one call, with no host read of a length.  Any pool and backend of this
package can use its rows.
"""

from __future__ import annotations

import torch

from qwenquest_amd import _lib
from qwenquest_amd.hisparse.coordinator import HiSparseCoordinator, pinned_zeros
from qwenquest_amd.memory import ReqToTokenPool

__all__ = ["BLOCK_TOKENS", "BlockReqToTokenPool", "CodedTokenToKVPool", "Fp4TokenToKVPool", "Fp8TokenToKVPool"]

BLOCK_TOKENS = 64

# what the device counts refused calls by, and what they are raised as
_REFUSALS = (
    (RuntimeError, "KV pool out of memory: too few free blocks for the batch"),
    (ValueError, "a request index or length lies outside the request table"),
    (ValueError, "a request is listed twice"),
    (ValueError, "the requests' tokens exceed total, or blocks are released that were not assigned"),
)


def _indexed(device: torch.device | str) -> torch.device:
    """``cuda`` as the device it stands for now: the pool's tensors lie there from now on."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return device


def _device_i64(t: torch.Tensor, device: torch.device, what: str) -> torch.Tensor:
    if t.dtype is torch.int64 and t.dim() == 1 and t.device == device and t.is_contiguous():
        return t
    if t.dim() != 1:
        raise ValueError(f"{what} must be one-dimensional, got {tuple(t.shape)}")
    if t.dtype.is_floating_point or t.dtype == torch.bool:
        raise ValueError(f"{what} must hold whole numbers, got {t.dtype}")
    return t.to(device=device, dtype=torch.int64).contiguous()


class BlockReqToTokenPool(ReqToTokenPool):
    """``ReqToTokenPool`` over ``num_blocks`` blocks of 64 pool rows (block 0 is padding).

    ``block_table [size, ceil(max_context_len / 64)]`` int32 lists a request's blocks (0: none),
    ``held [size]`` int32 counts them, ``free_blocks[: free_count]`` is the stack of free ones.
    A batch that cannot be served (too few blocks, a request or length outside its table, a
    request listed twice, more tokens than announced) is refused on the device as a whole: every
    row of its answer is the padding row 0, nothing is taken, and ``check_errors`` raises.
    Calls on one pool must not overlap on different streams.
    """

    def __init__(self, size: int, max_context_len: int, num_blocks: int, device: torch.device | str):
        super().__init__(size, max_context_len, _indexed(device))
        if self.device.type != "cuda":
            raise RuntimeError("qwenquest_amd.BlockReqToTokenPool needs a GPU device (no CPU path)")
        if not 1 <= num_blocks <= 1 << 24:
            raise ValueError(f"num_blocks must be at least 1 (the padding block) and at most 2^24, got {num_blocks}")
        if not 1 <= size <= 1 << 18 or not 1 <= max_context_len < 1 << 30:
            raise ValueError(f"at most 2^18 requests of under 2^30 tokens, got {size} of {max_context_len}")
        dev = self.device
        self.num_blocks = num_blocks
        self.max_blocks = (max_context_len + BLOCK_TOKENS - 1) // BLOCK_TOKENS
        self.block_table = torch.zeros((size, self.max_blocks), dtype=torch.int32, device=dev)
        self.held = torch.zeros(size, dtype=torch.int32, device=dev)
        self.free_blocks = torch.arange(num_blocks - 1, 0, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), num_blocks - 1, dtype=torch.int32, device=dev)
        # refused calls by reason, never set back; what has been raised of them
        self._err = torch.zeros(len(_REFUSALS), dtype=torch.int32, device=dev)
        self._raised = [0] * len(_REFUSALS)
        self._bind()

    def _bind(self) -> None:
        """The C entries' view of the pool, whose tensors stay where they are, and the counts' mirror."""
        self._err_host = pinned_zeros((len(_REFUSALS),), torch.int32)
        self._err_host.copy_(self._err)
        self._err_host_dev = HiSparseCoordinator._device_address(self._err_host)
        r2t, bt = self.req_to_token, self.block_table
        self._args = (_lib.ptr(bt), bt.stride(0), _lib.ptr(r2t), r2t.stride(0), r2t.shape[1], r2t.shape[0],
                      _lib.ptr(self.held), _lib.ptr(self.free_blocks), _lib.ptr(self.free_count), self.free_blocks.numel())

    def __getstate__(self) -> dict:  # addresses hold for this pool's own tensors, not for a copy's or a pickle's
        return {name: value for name, value in self.__dict__.items() if name not in ("_args", "_err_host", "_err_host_dev")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._bind()

    def available_blocks(self) -> int:
        """Free blocks (reads the device: a synchronisation)."""
        return int(self.free_count.item())

    def _workspace(self, bs: int) -> torch.Tensor:
        # of this call alone: a graph's replay must not find another call's plan in it
        need = int(_lib.load().qq_block_workspace_bytes(bs))
        return torch.empty(max(need, 1), dtype=torch.uint8, device=self.device)

    def _assign(self, rpi, lens, new_lens, total: int) -> tuple[torch.Tensor, torch.Tensor]:
        loc, pos = torch.empty((2, total), dtype=torch.int64, device=self.device).unbind(0)
        ws = self._workspace(rpi.numel()) if new_lens is not None else None
        with _lib.on(self.device):
            _lib.call(
                "qq_block_assign", _lib.ptr(rpi), _lib.ptr(lens), _lib.ptr(new_lens), int(rpi.numel()), total,
                *self._args, _lib.ptr(loc), _lib.ptr(pos), _lib.ptr(self._err), self._err_host_dev, _lib.ptr(ws),
                0 if ws is None else ws.numel(), _lib.stream(self.device),
            )
        return loc, pos

    def assign(self, req_pool_indices: torch.Tensor, prefix_lens: torch.Tensor, new_lens: torch.Tensor,
               total: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows and positions, ``[total]`` int64 each, of the next ``new_lens[i]`` tokens of each
        listed request behind its first ``prefix_lens[i]``, one request after the other; blocks it
        lacks are taken.  ``total`` is the batch's number of new tokens, as the caller's inputs
        have it; rows past the requests' tokens are 0.  A request without new tokens is ignored;
        asked again for the same lengths, the answer is the same."""
        rpi = _device_i64(req_pool_indices, self.device, "req_pool_indices")
        prefix = _device_i64(prefix_lens, self.device, "prefix_lens")
        new = _device_i64(new_lens, self.device, "new_lens")
        if not rpi.numel() == prefix.numel() == new.numel():
            raise ValueError("req_pool_indices, prefix_lens and new_lens differ in length")
        if total < 0:
            raise ValueError(f"total must not be negative, got {total}")
        return self._assign(rpi, prefix, new, int(total))

    def assign_decode(self, req_pool_indices: torch.Tensor, seq_lens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Row and position of each request's token at ``seq_lens[i] - 1``, ``[bs]`` int64 each, as
        a decode step needs them.  A padded entry has ``seq_lens[i] < 1`` and gets row 0."""
        rpi = _device_i64(req_pool_indices, self.device, "req_pool_indices")
        seq = _device_i64(seq_lens, self.device, "seq_lens")
        if rpi.numel() != seq.numel():
            raise ValueError("req_pool_indices and seq_lens differ in length")
        return self._assign(rpi, seq, None, int(rpi.numel()))

    def release(self, req_pool_indices: torch.Tensor) -> None:
        """Give the listed requests' blocks back and clear their tables."""
        rpi = _device_i64(req_pool_indices, self.device, "req_pool_indices")
        ws = self._workspace(rpi.numel())
        with _lib.on(self.device):
            _lib.call("qq_block_release", _lib.ptr(rpi), int(rpi.numel()), *self._args, _lib.ptr(self._err),
                      self._err_host_dev, _lib.ptr(ws), ws.numel(), _lib.stream(self.device))

    def free(self, req_pool_idx: int) -> None:
        """Release the request's blocks, then its slot (memory.py:44-50)."""
        self.release(torch.tensor([req_pool_idx], dtype=torch.int64))
        super().free(req_pool_idx)

    def check_errors(self, sync: bool = True) -> None:
        """Raise what calls since the last error were refused for on the device: ValueError for lengths,
        requests or totals that do not fit, RuntimeError when only the blocks ran out.  ``sync``:
        read the device's counts (a synchronisation with the current stream); otherwise their mirror in
        pinned host memory, which shows the calls whose kernels have finished.  A call that is
        refused meanwhile is raised by the next check."""
        counts = (self._err if sync else self._err_host).tolist()
        new = []
        for i, n in enumerate(counts):
            if 0 < (n - self._raised[i]) % (1 << 32) < 1 << 31:
                self._raised[i] = n
                new.append(_REFUSALS[i])
        if new:
            kind = ValueError if any(k is ValueError for k, _ in new) else RuntimeError
            raise kind("; ".join(said for _, said in new))

    def poll_errors(self) -> None:
        """``check_errors`` without a synchronisation, as a caller of replayed graphs needs it."""
        self.check_errors(sync=False)


class CodedTokenToKVPool:
    """What the pools of coded blocks share: per layer ``num_blocks`` blocks of 64 tokens (block 0 is padding)
    of codes (``k_codes``, ``v_codes [num_layers, num_blocks, kv_heads, ...]``, in the order that the attention
    kernels take them) and scales (``k_scale``, ``v_scale``).  ``set_kv_buffer`` writes values and
    ``get_rows`` reads them, by pool row.  ``head_dim`` 64 or 128."""

    #: the C entries' prefix
    kind: str = ""

    def __init__(self, num_blocks: int, num_layers: int, kv_heads: int, head_dim: int, device: torch.device | str):
        self.device = _indexed(device)
        if self.device.type != "cuda":
            raise RuntimeError(f"qwenquest_amd.{type(self).__name__} needs a GPU device (no CPU path)")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if not 1 <= num_blocks <= 1 << 24 or num_layers < 1 or not 1 <= kv_heads <= 1024:
            raise ValueError(f"num_blocks must be 1 .. 2^24, kv_heads 1 .. 1024 and num_layers at least 1, got {num_blocks}, "
                             f"{kv_heads} and {num_layers}")
        self.num_blocks = num_blocks
        self.num_layers = num_layers
        self.kv_heads = kv_heads
        self.head_dim = head_dim
        self.size = num_blocks * BLOCK_TOKENS - 1
        self._allocate((num_layers, num_blocks, kv_heads))
        self._bind()

    def _bind(self) -> None:
        """One layer's codes and scales with the geometry, as the C entries take them; the tensors stay where they are."""
        steps = [(_lib.ptr(t), t.stride(0) * t.element_size()) for t in (self.k_codes, self.v_codes, self.k_scale, self.v_scale)]
        self._layers = [(*(base + i * step for base, step in steps), self.num_blocks, self.kv_heads, self.head_dim)
                        for i in range(self.num_layers)]

    def __getstate__(self) -> dict:  # addresses hold for this pool's own tensors, not for a copy's or a pickle's
        return {name: value for name, value in self.__dict__.items() if name != "_layers"}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._bind()

    def _allocate(self, shape: tuple[int, int, int]) -> None:
        raise NotImplementedError

    @property
    def rows(self) -> int:
        return self.num_blocks * BLOCK_TOKENS

    def storage_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.v_codes, self.k_scale, self.v_scale))

    def layer_args(self, layer_id: int) -> tuple:
        """One layer's codes and scales with the geometry, as the C entries take them."""
        if not 0 <= layer_id < self.num_layers:
            raise IndexError(f"layer {layer_id} of {self.num_layers}")
        return self._layers[layer_id]

    def new_rows(self, k: torch.Tensor, v: torch.Tensor, n: int) -> tuple[torch.Tensor, torch.Tensor]:
        """``k`` and ``v`` of n tokens as the C entries take them: one bf16 or fp32 type, dense,
        16-byte aligned."""
        if k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float32):
            k, v = k.float(), v.float()
        out = []
        for x in (k, v):
            if x.numel() != n * self.kv_heads * self.head_dim:
                raise ValueError(f"expected {n} rows of {self.kv_heads} x {self.head_dim}, got {tuple(x.shape)}")
            if x.is_cuda and x.device != self.device:
                raise ValueError(f"k and v must lie on {self.device}, got {x.device}")
            if not x.is_contiguous():
                x = x.contiguous()
            out.append(x.clone() if x.data_ptr() % 16 else x)
        return out[0], out[1]

    def set_kv_buffer(self, layer_id: int, loc: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
        """Write ``k``/``v`` ``[n, kv_heads, head_dim]`` at rows ``loc`` (memory.py:114-120).  Rows of
        block 0 and outside the pool are skipped; the rows of one block stand next to each other in
        ``loc``, as a slot map has them."""
        _lib.refuse_tracing("a store into a pool of codes")
        loc = _device_i64(loc, self.device, "loc")
        n = int(loc.numel())
        if n == 0:
            return
        k, v = self.new_rows(k, v, n)
        with _lib.on(self.device):
            _lib.call(f"qq_{self.kind}_store", *self.layer_args(layer_id), _lib.ptr(k), _lib.ptr(v), _lib.dtype_code(k.dtype),
                      _lib.ptr(loc), n, _lib.stream(self.device))

    def get_rows(self, layer_id: int, loc: torch.Tensor,
                 dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """K and V values ``[n, kv_heads, head_dim]`` of rows ``loc``: exact in bf16 (and fp32); NaN
        for a row outside the pool."""
        _lib.refuse_tracing("rows out of a pool of codes")
        code = _lib.dtype_code(dtype)
        loc = _device_i64(loc, self.device, "loc")
        n = int(loc.numel())
        k, v = torch.empty((2, n, self.kv_heads, self.head_dim), dtype=dtype, device=self.device).unbind(0)
        if n:
            with _lib.on(self.device):
                _lib.call(f"qq_{self.kind}_rows", *self.layer_args(layer_id), _lib.ptr(loc), n, _lib.ptr(k), _lib.ptr(v), code,
                          _lib.stream(self.device))
        return k, v


class Fp8TokenToKVPool(CodedTokenToKVPool):
    """A K/V pool in 8 bits: per layer ``num_blocks`` blocks of 64 tokens (block 0 is padding) of
    e4m3 codes, with one power-of-two float scale for each block and KV head, K and V apart
    (``k_scale``, ``v_scale`` ``[num_layers, num_blocks, kv_heads]``).  ``head_dim`` 64 or 128.

    The codes (``k_codes``, ``v_codes``) lie in the order that the attention kernels take them;
    ``set_kv_buffer`` writes values and ``get_rows`` reads them, by pool row.  Of a block's values
    the scale is the least power of two (not under 2^-110) that keeps them within the codes' 448;
    a later token with a larger value raises it, and the block's earlier codes are rounded again.
    Writing a block's first row begins the block: what it held is gone.  Values that are not finite
    make the scale of their (block, head) NaN until the block is begun again, and whoever attends
    it gets NaN.
    """

    dtype = torch.float8_e4m3fn

    kind = "fp8"

    def _allocate(self, shape):
        codes = (*shape, BLOCK_TOKENS * self.head_dim)
        self.k_codes = torch.zeros(codes, dtype=torch.uint8, device=self.device)
        self.v_codes = torch.zeros(codes, dtype=torch.uint8, device=self.device)
        self.k_scale = torch.full(shape, 2.0**-110, dtype=torch.float32, device=self.device)
        self.v_scale = torch.full(shape, 2.0**-110, dtype=torch.float32, device=self.device)


class Fp4TokenToKVPool(CodedTokenToKVPool):
    """A K/V pool in 4 bits: per layer ``num_blocks`` blocks of 64 tokens (block 0 is padding) of e2m1
    codes with power-of-two scales, each the byte of its exponent: of K one for each token, KV head and 32
    channels (``k_scale [num_layers, num_blocks, kv_heads, 2 * head_dim]``), of V one for each token and KV head
    (``v_scale [num_layers, num_blocks, kv_heads, 64]``).  ``head_dim`` 64 or 128.  133 bytes for a token's K and V of
    128 channels, where bf16 takes 512.

    Of the values that share a scale it is the least power of two that keeps them within 7 times itself
    (values between 6 and 7 times it become 6 times it, the largest code), for K 2^-96 at least (and 2^125 at
    most), for V 2^-50.  Tokens are independent of each other: a row may be written at any time and over and
    over.  Of a token and KV head whose K or V holds a value that is not finite, or whose V one above 7 * 2^59,
    nothing is kept: K and V read back as NaN, and whoever attends it gets NaN.
    """

    kind = "fp4"
    #: two e2m1 codes a byte
    dtype = torch.uint8

    def _allocate(self, shape):
        codes = (*shape, BLOCK_TOKENS * self.head_dim // 2)
        self.k_codes = torch.zeros(codes, dtype=torch.uint8, device=self.device)
        self.v_codes = torch.zeros(codes, dtype=torch.uint8, device=self.device)
        self.k_scale = torch.full((*shape, 2 * self.head_dim), 127, dtype=torch.uint8, device=self.device)
        self.v_scale = torch.full((*shape, BLOCK_TOKENS), 127, dtype=torch.uint8, device=self.device)
