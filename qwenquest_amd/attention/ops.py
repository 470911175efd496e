"""Attention math (reference ``src/qwenquest/attention/ops.py``).

``decode_attention`` runs the HIP split-K kernel over an explicit row list;
``fp8_decode_attention`` and ``fp8_extend_attention`` run the HIP kernels over an 8-bit block cache;
``extend_attention_batch`` runs a whole prefill batch (bf16, head_dim 128) in the HIP
prefill kernel; ``extend_attention``, one request of any shape, uses torch's SDPA on the
device, in float32.
"""

from __future__ import annotations

from typing import TYPE_CHECKING

import torch
import torch.nn.functional as F

from qwenquest_amd import _lib
from qwenquest_amd.batch import DecodePlan

if TYPE_CHECKING:
    from qwenquest_amd.paged import Fp8TokenToKVPool
    from qwenquest_amd.quest import QuestAlgorithm

__all__ = ["decode_attention", "extend_attention", "extend_attention_batch", "fp8_decode_attention",
           "fp8_extend_attention", "fp8_quest_step", "AttentionWorkspace"]


class AttentionWorkspace:
    """Device workspace of the split-K attention kernels (per-chunk (m, l, o) partials)."""

    def __init__(self, device: torch.device):
        self.device = device
        self.buf = torch.empty(0, dtype=torch.uint8, device=device)

    def get(self, bs: int, max_rows: int, heads: int, head_dim: int) -> torch.Tensor:
        need = int(_lib.load().qq_decode_attention_workspace_bytes(bs, max_rows, heads, head_dim))
        if self.buf.numel() < need:
            self.buf = torch.empty(need, dtype=torch.uint8, device=self.device)
        return self.buf


_workspaces: dict[torch.device, AttentionWorkspace] = {}


def _workspace(device: torch.device) -> AttentionWorkspace:
    ws = _workspaces.get(device)
    if ws is None:
        ws = _workspaces[device] = AttentionWorkspace(device)
    return ws


def decode_attention_rows(
    q: torch.Tensor,
    k_buf: torch.Tensor,
    v_buf: torch.Tensor,
    rows: torch.Tensor,
    actual_lens: torch.Tensor,
    scaling: float,
    *,
    workspace: AttentionWorkspace | None = None,
    out: torch.Tensor | None = None,
    sync: torch.Tensor | None = None,
) -> torch.Tensor:
    """Batched form: request ``i`` attends ``q[i] [H, D]`` over ``k_buf[rows[i, :actual_lens[i]]]``.

    ``rows`` ``[bs, >= max(actual_lens)]`` int64, ``k_buf``/``v_buf`` ``[rows, KV, D]``.
    Returns ``[bs, H*D]`` in q's dtype.  With ``sync`` (a zeroed uint8 buffer of at least
    ``qq_quest_layer_step_sync_bytes`` bytes) the bf16 shapes with D = 128 and 1, 2, 4 or 8
    KV heads run the attention kernel of the fused Quest layer step, whose arithmetic
    QuestHiSparseBackend shares with QuestOnlyBackend.
    """
    bs, heads, dim = q.shape
    kv = k_buf.shape[1]
    q = q.contiguous()
    rows = rows.to(torch.int64).contiguous()
    actual = actual_lens.to(device=q.device, dtype=torch.int32).contiguous()
    ws = workspace or _workspace(q.device)
    buf = ws.get(bs, rows.shape[1], heads, dim)
    res = out if out is not None else torch.empty((bs, heads * dim), dtype=q.dtype, device=q.device)
    _lib.call(
        "qq_decode_attention_rows", _lib.ptr(q), _lib.dtype_code(q.dtype), q.stride(0), heads,
        _lib.ptr(k_buf), _lib.ptr(v_buf), _lib.dtype_code(k_buf.dtype), k_buf.shape[0], kv, dim,
        _lib.ptr(rows), rows.stride(0), _lib.ptr(actual), bs, float(scaling), _lib.ptr(res),
        _lib.ptr(buf), buf.numel(), _lib.ptr(sync) if sync is not None else None,
        sync.numel() if sync is not None else 0, _lib.stream(q.device),
    )
    return res


def decode_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scaling: float) -> torch.Tensor:
    """One query ``[H, D]`` against the listed rows ``k, v [n, KV, D]`` -> ``[H*D]``
    (reference ops.py:48-66; duplicates counted, fp32 softmax and accumulation)."""
    n = k.shape[0]
    k = k.to(v.dtype).contiguous()
    v = v.contiguous()
    rows = torch.arange(n, dtype=torch.int64, device=q.device).unsqueeze(0)
    actual = torch.full((1,), n, dtype=torch.int32, device=q.device)
    return decode_attention_rows(q.unsqueeze(0), k, v, rows, actual, scaling)[0]


def extend_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prefix_len: int, scaling: float) -> torch.Tensor:
    """Dense causal prefill of one request (reference ops.py:18-45), torch SDPA in float32."""
    n, num_heads, head_dim = q.shape
    kv_len, kv_heads, _ = k.shape
    group = num_heads // kv_heads
    qh = q.float().transpose(0, 1).unsqueeze(0)
    kh = k.float().repeat_interleave(group, dim=1).transpose(0, 1).unsqueeze(0).contiguous()
    vh = v.float().repeat_interleave(group, dim=1).transpose(0, 1).unsqueeze(0).contiguous()
    q_pos = prefix_len + torch.arange(n, device=q.device)
    mask = torch.arange(kv_len, device=q.device).unsqueeze(0) <= q_pos.unsqueeze(1)
    out = F.scaled_dot_product_attention(qh.contiguous(), kh, vh, attn_mask=mask, scale=scaling)
    return out[0].transpose(0, 1).reshape(n, num_heads * head_dim).to(q.dtype)


# Pinned words for the verdicts of checked prefill launches, as many as calls were ever in
# flight at once (one per thread): each is taken for one call and is back when the call has read
# it.  After an error the device may still write its word: it is not used again.
_verdicts: list = []


def _extend_launch(
    q: torch.Tensor,
    k_buf: torch.Tensor,
    v_buf: torch.Tensor,
    req_to_token: torch.Tensor,
    lens: tuple[torch.Tensor, ...],
    scaling: float,
    checked: bool,
) -> tuple[torch.Tensor, int | None]:
    """qq_extend_attention; the output, and the verdict on the lengths if asked for."""
    n, heads, dim = q.shape
    kv, bs, dev = k_buf.shape[1], int(lens[0].shape[0]), q.device
    q = q.contiguous()
    if q.data_ptr() % 16:  # the kernel reads 16-byte pieces
        q = q.clone()
    rpi, seq, prefix, ext = (
        t if t.dtype == torch.int64 and t.device == dev and t.is_contiguous()
        else t.to(device=dev, dtype=torch.int64).contiguous() for t in lens)
    width, stride = req_to_token.shape[1], req_to_token.stride(0)
    if stride != width:  # columns of a wider table: the kernel cuts a context at the stride
        seq = seq.clamp(max=width)
    need = int(_lib.load().qq_extend_attention_workspace_bytes(n, bs, heads, kv, stride))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    out = torch.empty((n, heads * dim), dtype=q.dtype, device=dev)
    args = (
        _lib.ptr(q), heads, _lib.ptr(k_buf), _lib.ptr(v_buf), k_buf.shape[0], kv, dim,
        _lib.ptr(req_to_token), stride, req_to_token.shape[0], _lib.ptr(rpi), _lib.ptr(seq),
        _lib.ptr(prefix), _lib.ptr(ext), bs, n, float(scaling), _lib.ptr(out), _lib.ptr(ws), need,
    )
    stream = _lib.stream(dev)
    if not checked:
        _lib.call("qq_extend_attention", *args, stream)
        return out, None
    try:
        verdict = _verdicts.pop()
    except IndexError:
        verdict = torch.empty(1, dtype=torch.int64, pin_memory=True).numpy()
    _lib.call("qq_extend_attention_checked", *args, verdict.ctypes.data, stream)
    found = int(verdict[0])
    _verdicts.append(verdict)
    return out, found


def extend_attention_batch(
    q: torch.Tensor,
    k_buf: torch.Tensor,
    v_buf: torch.Tensor,
    req_to_token: torch.Tensor,
    req_pool_indices: torch.Tensor,
    seq_lens: torch.Tensor,
    prefix_lens: torch.Tensor,
    extend_lens: torch.Tensor,
    scaling: float,
) -> torch.Tensor:
    """Dense causal prefill of a batch (the loop of base.py:65-93): ``q [n, H, 128]`` holds the
    requests' new tokens one request after the other, ``k_buf``/``v_buf [rows, KV, 128]`` the
    pool with the new K/V in it.  bf16; returns ``[n, H*128]``.  The lengths (each ``[>= bs]``)
    are read on the device only; a request whose index lies outside the table gets NaN, as do
    rows of q past the requests' tokens."""
    lens = (req_pool_indices, seq_lens, prefix_lens, extend_lens)
    return _extend_launch(q, k_buf, v_buf, req_to_token, lens, scaling, False)[0]


def extend_attention_batch_checked(
    q: torch.Tensor,
    k_buf: torch.Tensor,
    v_buf: torch.Tensor,
    req_to_token: torch.Tensor,
    req_pool_indices: torch.Tensor,
    seq_lens: torch.Tensor,
    prefix_lens: torch.Tensor,
    extend_lens: torch.Tensor,
    scaling: float,
) -> torch.Tensor | None:
    """``extend_attention_batch`` outside a graph capture: the requests' rows only, and None for a
    batch that the loop treats in another way (or refuses).

    The launch looks at the lengths as it begins and the host waits for that, not for its end: the
    device is not left idle, and no copy, event or launch is queued (600 new tokens 30 us, 29
    without a verdict; by a launch of its own 40, with an event 43, by a copy of the lengths 52)."""
    lens = (req_pool_indices, seq_lens, prefix_lens, extend_lens)
    out, verdict = _extend_launch(q, k_buf, v_buf, req_to_token, lens, scaling, True)
    if verdict == 1:
        return None
    tokens = verdict // 2
    return out if tokens >= out.shape[0] else out[:tokens]


def _lengths(t: torch.Tensor, n: int, device: torch.device, what: str) -> torch.Tensor:
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what} must have {n} entries, got {tuple(t.shape)}")
    if t.dtype == torch.int64 and t.device == device and t.is_contiguous():
        return t
    return t.to(device=device, dtype=torch.int64).contiguous()


def _queries(q: torch.Tensor, pool: Fp8TokenToKVPool) -> torch.Tensor:
    """``q [n, H, D]`` (or ``[n, H*D]``) dense and 16-byte aligned."""
    dim = pool.head_dim
    if q.device != pool.device:
        raise ValueError(f"q lies on {q.device}, the pool on {pool.device}")
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"unsupported dtype {q.dtype}; the kernels take bfloat16 or float32")
    if q.dim() == 2 and q.shape[1] % dim == 0:
        q = q.reshape(q.shape[0], q.shape[1] // dim, dim)
    if q.dim() != 3 or q.shape[2] != dim:
        raise ValueError(f"queries must be [n, heads, {dim}], got {tuple(q.shape)}")
    if q.shape[1] == 0 or q.shape[1] % pool.kv_heads:
        raise ValueError(f"q_heads {q.shape[1]} not divisible by kv_heads {pool.kv_heads}")
    q = q.detach().contiguous()
    return q.clone() if q.data_ptr() % 16 else q


def fp8_decode_plan(pool: Fp8TokenToKVPool, block_table: torch.Tensor, req_pool_indices: torch.Tensor,
                    seq_lens: torch.Tensor) -> DecodePlan:
    """What ``fp8_decode_attention`` over whole contexts makes of a step's lengths, once for the step's
    layers, on the current stream."""
    dev = pool.device
    bs = int(req_pool_indices.shape[0])
    table = _lib.table_args(block_table, dev)
    rpi = _lengths(req_pool_indices, bs, dev, "req_pool_indices")
    seq = _lengths(seq_lens, bs, dev, "seq_lens")
    need = int(_lib.load().qq_fp8_decode_workspace_bytes(bs, pool.kv_heads, pool.kv_heads, pool.head_dim))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    stream = _lib.stream(dev)
    with _lib.on(dev):
        _lib.call("qq_fp8_decode_plan", pool.num_blocks, pool.kv_heads, pool.head_dim, table[2], table[3],
                  _lib.ptr(rpi), _lib.ptr(seq), bs, _lib.ptr(ws), need, stream)
    return DecodePlan(bs, ws, stream, _lib.capture_id(dev, stream))


def fp8_decode_attention(
    q: torch.Tensor,
    pool: Fp8TokenToKVPool,
    layer_id: int,
    block_table: torch.Tensor,
    req_pool_indices: torch.Tensor,
    seq_lens: torch.Tensor,
    scaling: float,
    *,
    positions: torch.Tensor | None = None,
    top_k: int = 0,
    new: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
    plan: DecodePlan | None = None,
) -> torch.Tensor:
    """Decode over an 8-bit pool: request ``i`` attends ``q[i] [H, D]`` over its first ``seq_lens[i]``
    tokens in the blocks ``block_table[req_pool_indices[i]]``, or, with ``positions [bs, >= top_k]``
    (``QuestAlgorithm.retrieve_topk``) and a longer context than ``top_k``, over the pages listed
    there and the last 64 tokens.  ``new``: ``(loc, k, v)`` of the batch's new tokens, stored first.
    ``plan``: this step's ``fp8_decode_plan`` (of the same pool, table, requests and lengths, on the
    same stream; not with ``positions``): up to 16 query heads per KV head then run as one launch,
    for which each new token lies in the last block of its own request's context and no two in one
    block (rows of block 0, the padding, aside); on another stream, or where the two calls are not in
    the same graph capture or both in none, they run as without it.
    Returns ``[bs, H*D]`` in q's dtype (bf16 or fp32): zeros for an empty context, NaN for a request
    outside the table or a context past its blocks."""
    dev = pool.device
    q = _queries(q, pool)
    bs, heads, dim = q.shape
    table = _lib.table_args(block_table, dev)
    rpi = _lengths(req_pool_indices, bs, dev, "req_pool_indices")
    seq = _lengths(seq_lens, bs, dev, "seq_lens")
    if positions is not None:
        if (positions.dim() != 2 or positions.dtype != torch.int32 or positions.device != dev
                or positions.shape[0] < bs or positions.shape[1] < top_k or positions.stride(1) != 1):
            raise ValueError(f"positions must be an int32 tensor [>= {bs}, >= {top_k}] on {dev}")
    loc = kn = vn = None
    if new is not None:
        loc = _lengths(new[0], bs, dev, "out_cache_loc")
        kn, vn = pool.new_rows(new[1], new[2], bs)
    out = torch.empty((bs, heads * dim), dtype=q.dtype, device=dev)
    if plan is not None and positions is not None:
        raise ValueError("a plan is of whole contexts, not of selected pages")
    need = int(_lib.load().qq_fp8_decode_workspace_bytes(bs, heads, pool.kv_heads, dim))
    stream = _lib.stream(dev)
    if plan is not None and heads <= 16 * pool.kv_heads and plan.usable(stream):
        ws = plan.workspace
        if plan.bs != bs or plan.top_k != 0 or ws.device != dev or ws.numel() != max(need, 1):
            raise ValueError("plan is not fp8_decode_plan's of this batch and pool")
    else:
        # of this call alone: it holds the division of the batch, which a graph's replay or a call on
        # another stream must not find replaced
        ws, plan = torch.empty(max(need, 1), dtype=torch.uint8, device=dev), None
    with _lib.on(dev):
        _lib.call(
            "qq_fp8_decode_attention", _lib.ptr(q), _lib.dtype_code(q.dtype), q.stride(0), heads, _lib.ptr(kn),
            _lib.ptr(vn), _lib.DTYPE_BF16 if kn is None else _lib.dtype_code(kn.dtype), _lib.ptr(loc),
            *pool.layer_args(layer_id), *table, _lib.ptr(rpi), _lib.ptr(seq), bs, _lib.ptr(positions),
            0 if positions is None else max(positions.stride(0), positions.shape[1]), int(top_k), float(scaling),
            _lib.ptr(out), _lib.ptr(ws), need, int(plan is not None), stream,
        )
    return out


def fp8_quest_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    loc: torch.Tensor,
    pool: Fp8TokenToKVPool,
    layer_id: int,
    block_table: torch.Tensor,
    quest: QuestAlgorithm,
    req_pool_indices: torch.Tensor,
    positions: torch.Tensor,
    scaling: float,
    phase: int = 3,
) -> torch.Tensor:
    """One layer of Quest decode over an 8-bit pool, after ``quest.decode_step_blocks``: the new tokens
    ``k``/``v`` go to rows ``loc``, the page scores select (``positions [>= bs, top_k]`` int32 is
    written, as ``QuestAlgorithm.retrieve_topk`` writes it), and ``q [bs, H, D]`` attends the selected
    pages.  On the stream of ``decode_step_blocks``, both in the same graph capture or in none, the
    step's division of the work saves a launch; each new token lies in the last block of its own
    request's context and no two in one block (rows of block 0 aside).  ``phase``: 1 = scoring and selection, 2 = store and attention after phase 1, 3 = both.
    Returns ``[bs, H*D]`` (complete after phase 2)."""
    dev, step = pool.device, quest._step
    if step is None:
        raise RuntimeError("decode_step_blocks() must be called once per decode step first")
    q = _queries(q, pool)
    bs, heads, dim = q.shape
    if step.seq_lens.shape[0] != bs:
        raise ValueError("batch size differs from the one given to decode_step_blocks()")
    if bs > quest.max_reqs:
        raise ValueError(f"batch {bs} exceeds max_reqs {quest.max_reqs}")
    if (quest.page_size != 64 or quest.kv_heads != pool.kv_heads or quest.head_dim != dim
            or quest.page_k_bounds.device != dev):
        raise ValueError("the Quest state is not of this pool's pages and heads")
    if not quest.start_layer <= layer_id < quest.end_layer:
        raise IndexError(f"layer {layer_id} is no Quest layer ({quest.start_layer} .. {quest.end_layer - 1})")
    if (positions.dtype != torch.int32 or positions.device != dev or not positions.is_contiguous()
            or positions.dim() != 2 or positions.shape[0] < bs or positions.shape[1] != quest.top_k):
        raise ValueError(f"positions must be a contiguous int32 tensor [>= {bs}, {quest.top_k}] on {dev}")
    table = _lib.table_args(block_table, dev)
    rpi = _lengths(req_pool_indices, bs, dev, "req_pool_indices")
    loc = _lengths(loc, bs, dev, "out_cache_loc")
    kn, vn = pool.new_rows(k, v, bs)
    out = torch.empty((bs, heads * dim), dtype=q.dtype, device=dev)
    need = int(_lib.load().qq_fp8_decode_workspace_bytes(bs, heads, pool.kv_heads, dim))
    stream = _lib.stream(dev)
    planned = step.plan is not None and heads <= 16 * pool.kv_heads and step.plan.usable(stream)
    ws = step.plan.workspace if planned else torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    if planned and (step.plan.bs != bs or step.plan.top_k != quest.top_k or ws.device != dev or ws.numel() != max(need, 1)):
        raise ValueError("the step's plan is not decode_step_blocks' of this batch and pool")
    with _lib.on(dev):
        _lib.call(
            "qq_fp8_quest_step", _lib.ptr(q), _lib.dtype_code(q.dtype), q.stride(0), heads, _lib.ptr(kn), _lib.ptr(vn),
            _lib.dtype_code(kn.dtype), _lib.ptr(loc), *pool.layer_args(layer_id), *table,
            _lib.ptr(quest.page_k_bounds), layer_id - quest.start_layer, _lib.ptr(rpi), _lib.ptr(step.seq_lens),
            _lib.ptr(step.candidate_limit_i32), bs, quest.max_reqs, quest.max_pages_per_req, quest.top_k, float(scaling),
            _lib.ptr(quest._scores_ws), _lib.ptr(positions), _lib.ptr(out), _lib.ptr(ws), need, int(phase), int(planned),
            stream,
        )
    return out


def fp8_extend_attention(
    q: torch.Tensor,
    pool: Fp8TokenToKVPool,
    layer_id: int,
    block_table: torch.Tensor,
    req_pool_indices: torch.Tensor,
    seq_lens: torch.Tensor,
    prefix_lens: torch.Tensor,
    extend_lens: torch.Tensor,
    scaling: float,
) -> torch.Tensor:
    """Causal prefill of a batch over an 8-bit pool that holds the new K/V: ``q [n, H, D]`` (bf16)
    holds the requests' new tokens one request after the other; token ``t`` of request ``i`` attends
    positions ``0 .. prefix_lens[i] + t``.  Returns ``[n, H*D]``; the lengths are read on the device
    only.  NaN: a request outside the table, a query tile that attends a block which is not there,
    rows of q past the requests' tokens."""
    dev = pool.device
    if q.dtype != torch.bfloat16:
        raise ValueError(f"unsupported dtype {q.dtype}; the prefill kernel takes bfloat16")
    q = _queries(q, pool)
    n, heads, dim = q.shape
    table = _lib.table_args(block_table, dev)
    bs = int(req_pool_indices.shape[0])
    rpi, seq, prefix, ext = (_lengths(t, bs, dev, what) for t, what in (
        (req_pool_indices, "req_pool_indices"), (seq_lens, "seq_lens"), (prefix_lens, "prefix_lens"),
        (extend_lens, "extend_lens")))
    if bs == 0 and n:
        raise ValueError(f"{n} tokens of no request")
    need = int(_lib.load().qq_fp8_extend_workspace_bytes(n, bs, heads, pool.kv_heads, dim, table[3]))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    out = torch.empty((n, heads * dim), dtype=q.dtype, device=dev)
    with _lib.on(dev):
        _lib.call(
            "qq_fp8_extend_attention", _lib.ptr(q), heads, *pool.layer_args(layer_id), *table, _lib.ptr(rpi),
            _lib.ptr(seq), _lib.ptr(prefix), _lib.ptr(ext), bs, n, float(scaling), _lib.ptr(out), _lib.ptr(ws), need,
            _lib.stream(dev),
        )
    return out
