"""Prefill attention over the 8-bit block cache against float64 over the cache's exact values; the
tolerance is half a step of the bf16 output, 0.64 * 2^-10 of the weights (the kernel's rounding of
them, here 2^-10), and the scores' float32 sums."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qwenquest_amd.attention.ops import fp8_extend_attention
from tests.test_gpu_fp8_decode import Setup, i64

pytestmark = pytest.mark.gpu


def check(s, out, q, prefix, new, scale, rows=None):
    """Every token's output, request by request (rows: the table row of each)."""
    G = q.shape[1] // s.kv
    assert out.shape == (q.shape[0], q.shape[1] * s.dim) and out.dtype == torch.bfloat16
    got, at = out.double().view(q.shape), 0
    for i, (p, n) in enumerate(zip(prefix, new)):
        r = i if rows is None else rows[i]
        k, v = (x.double() for x in s.pool.get_rows(s.layer, s.rows(r, np.arange(p + n)), torch.float32))
        seen = torch.arange(p + n, device=s.dev)[None] <= p + torch.arange(n, device=s.dev)[:, None]
        for h in range(q.shape[1] if n else 0):
            qh, kh, vh = q[at : at + n, h].double(), k[:, h // G].contiguous(), v[:, h // G].contiguous()
            t = (qh @ kh.T.contiguous() * scale).masked_fill(~seen, -np.inf)
            w = torch.softmax(t, -1)
            want, spread = w @ vh, w @ vh.abs()
            size = ((qh.abs() @ kh.abs().T.contiguous()) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            rel = 2.0**-10 + 2 * (s.dim + 4) * 2.0**-23 * size + (p + n) * 2.0**-23
            err = (got[at : at + n, h] - want).abs() / (2.0**-8 * want.abs() + rel * spread + 1e-38)
            assert (err <= 1).all(), f"request {i} head {h}: off by {err.max().item():.2f} tolerances at {err.argmax().item()}"
        at += n


def batch(cuda, prefix, new, kv, dim, heads, seed=0, pad=0, **kw):
    s = Setup(cuda, [p + n for p, n in zip(prefix, new)], kv, dim, seed=seed, **kw)
    q = s.queries(heads, torch.bfloat16, seed, n=sum(new) + pad)
    lens = (torch.arange(len(new)), i64([p + n for p, n in zip(prefix, new)], cuda), i64(prefix, cuda), i64(new, cuda))
    return s, q, lens


@pytest.mark.parametrize("heads, kv, dim", [(32, 4, 128), (1, 1, 128), (3, 1, 64), (48, 1, 128), (8, 8, 64), (10, 2, 128), (7, 1, 64)])
def test_ragged_batches(cuda, heads, kv, dim):
    prefix, new = [0, 63, 64, 200, 0, 1, 500, 65], [1, 1, 65, 130, 0, 64, 33, 300]
    s, q, lens = batch(cuda, prefix, new, kv, dim, heads, seed=heads)
    out = fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, dim**-0.5)
    check(s, out, q, prefix, new, dim**-0.5)


@pytest.mark.parametrize("prefix, new", [([8192], [8]), ([4000, 0, 2500], [3, 1, 40]), ([20000], [1]), ([0], [700]), ([5000], [100])])
def test_splits_of_long_contexts(cuda, prefix, new):
    """Few query rows before many tokens: the context divided over blocks, and merged."""
    for dim in (64, 128):
        s, q, lens = batch(cuda, prefix, new, 2, dim, 8, seed=len(new) + dim)
        out = fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1)
        check(s, out, q, prefix, new, 0.1)
        assert torch.equal(out, fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1))


def test_many_requests(cuda):
    new = [1 + i % 7 for i in range(150)]
    prefix = [(37 * i) % 200 for i in range(150)]
    s, q, lens = batch(cuda, prefix, new, 2, 64, 4)
    check(s, fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1), q, prefix, new, 0.1)


@pytest.mark.parametrize("scale", [1e-30, 3.0])
def test_small_and_large_scales(cuda, scale):
    s, q, lens = batch(cuda, [100], [90], 1, 128, 4)
    check(s, fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, scale), q, [100], [90], scale)


def test_values_of_very_different_size(cuda):
    """Blocks whose V scales lie 2^30 and more apart, a block of zeros among them, in rising and falling
    order: a weight is lost only next to values that are larger by far more than a bf16 holds."""
    prefix, new = [0, 0, 64], [330, 330, 300]
    s, q, lens = batch(cuda, prefix, new, 1, 128, 4, seed=3)
    gen = torch.Generator(device=cuda).manual_seed(1)
    for r, sizes in enumerate(([0, 1, 2.0**-12, 2.0**10, 1, 1], [2.0**25, 2.0**5, 0, 1, 2.0**-20, 1], [2.0**-60, 0, 2.0**-55, 1, 2.0**60, 1])):
        for b, size in enumerate(sizes):
            x = torch.empty((64, 1, 128), device=cuda).normal_(generator=gen)
            s.pool.set_kv_buffer(s.layer, s.rows(r, np.arange(b * 64, b * 64 + 64)), x, x * size)
    check(s, fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1), q, prefix, new, 0.1)


@pytest.mark.parametrize("prefix, new", [([0], [200]), ([2000], [3])])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("large", [1.0, 4.0, 16.0, 64.0])
def test_a_channel_that_carries_the_scores(cuda, large, dim, prefix, new):
    """One channel in which every key is large: what tells tokens apart are the others' products, next to one
    that is up to 2^16 times theirs.  The tolerance is that of sums in float32."""
    s, q, lens = batch(cuda, prefix, new, 1, dim, 4, seed=6)
    gen = torch.Generator(device=cuda).manual_seed(3)
    n = prefix[0] + new[0]
    k = torch.empty((n, 1, dim), device=cuda).normal_(generator=gen) * 0.5
    k[..., 0] = large
    s.pool.set_kv_buffer(s.layer, s.rows(0, np.arange(n)), k, torch.empty((n, 1, dim), device=cuda).normal_(generator=gen))
    q[..., 0] = large
    check(s, fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.25), q, prefix, new, 0.25)


@pytest.mark.parametrize("prefix, new", [([0], [330]), ([2000], [3]), ([60, 0], [270, 200])])
@pytest.mark.parametrize("size", [2.0**20, 2.0**40, 2.0**-40])
@pytest.mark.parametrize("at", [0, 2, -1])
def test_values_of_very_different_size_and_weight(cuda, prefix, new, size, at):
    """One block whose values are far larger (or smaller) than the others' and whose tokens weigh next to
    nothing, 2^-90: the others' values come back as without it."""
    dim, scale = 64, 0.5
    s, q, lens = batch(cuda, prefix, new, 1, dim, 4, seed=5)
    gen = torch.Generator(device=cuda).manual_seed(2)
    q.mul_(0.25)
    q[..., 0] = 8.0
    for r, (p, n) in enumerate(zip(prefix, new)):
        blocks = -(-(p + n) // 64)
        for b in range(blocks):
            k = torch.empty((64, 1, dim), device=cuda).normal_(generator=gen) * 0.25
            v = torch.empty((64, 1, dim), device=cuda).normal_(generator=gen)
            odd = b == at % blocks
            k[..., 0] = -8.0 if odd else 8.0
            s.pool.set_kv_buffer(s.layer, s.rows(r, np.arange(b * 64, b * 64 + 64)), k, v * (size if odd else 1.0))
    check(s, fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, scale), q, prefix, new, scale)


def test_extreme_key_scales(cuda):
    s, q, lens = batch(cuda, [0], [200], 1, 64, 2)
    for b, size in enumerate((1e-33, 1.0, 0.0)):
        x = torch.randn((64, 1, 64), device=cuda)
        s.pool.set_kv_buffer(s.layer, s.rows(0, np.arange(b * 64, b * 64 + 64)), x * size, x)
    check(s, fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.3), q, [0], [200], 0.3)


def test_rows_and_requests_that_are_not_there(cuda):
    prefix, new = [100, 0, 30], [70, 129, 65]
    s, q, lens = batch(cuda, prefix, new, 2, 128, 6, pad=37)
    out = fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1)
    check(s, out[: sum(new)], q[: sum(new)], prefix, new, 0.1)
    assert out[sum(new) :].isnan().all()
    rpi = i64([0, 3, -1], cuda)  # outside the table; the last row, from its end
    out = fp8_extend_attention(q, s.pool, s.layer, s.table, rpi, *lens[1:], 0.1)
    assert out[70:199].isnan().all() and not out[:70].isnan().any() and not out[199 : sum(new)].isnan().any()
    same = fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1)
    assert torch.equal(out[:70], same[:70]) and torch.equal(out[199 : sum(new)], same[199 : sum(new)])
    # a block that is not there: the query tiles that attend it
    table = s.table.clone()
    table[1, 2] = 0
    out = fp8_extend_attention(q, s.pool, s.layer, table, *lens, 0.1).view(-1, 6, 128)
    assert out[70 + 128].isnan().all() and torch.equal(out[:70].reshape(70, -1), same[:70])
    assert torch.equal(out[70 : 70 + 42].reshape(42, -1), same[70 : 70 + 42])  # the first tile: 128 rows of 3 heads
    # fewer rows of q than tokens: the last request's are cut
    out = fp8_extend_attention(q[:200], s.pool, s.layer, s.table, *lens, 0.1)
    assert torch.equal(out, same[:200])
    # lengths of no sense attend nothing
    out = fp8_extend_attention(q, s.pool, s.layer, s.table, lens[0], i64([-5, 129, 1 << 50], cuda), i64([100, 0, -(1 << 50)], cuda), lens[3], 0.1)
    assert out[:70].isnan().all() and torch.equal(out[70:199], same[70:199]) and out[199 : sum(new)].isnan().all()


def test_spoilt_values_reach_those_who_attend_them(cuda):
    """A value that is not finite spoils its (block, head): rows before the block have their answers."""
    prefix, new = [0, 64], [300, 200]
    s, q, lens = batch(cuda, prefix, new, 2, 64, 4)
    clean = fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1).view(-1, 4, 64)
    x = [torch.randn(1, 2, 64, device=cuda) for _ in range(2)]
    x[0][0, 0, 5] = float("nan")
    s.pool.set_kv_buffer(s.layer, s.rows(0, [150]), *x)
    y = [torch.randn(1, 2, 64, device=cuda) for _ in range(2)]
    y[1][0, 1, 9] = float("inf")
    s.pool.set_kv_buffer(s.layer, s.rows(1, [200]), *y)
    out = fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1).view(-1, 4, 64)
    assert torch.equal(out[:128], clean[:128]) and out[128:300, :2].isnan().all() and not out[128:300, 2:].isnan().any()
    at = 300 + 192 - 64
    assert torch.equal(out[300:at, 2:], clean[300:at, 2:]) and out[at:, 2:].isnan().all() and not out[at:, :2].isnan().any()


def test_queries_that_are_not_finite(cuda):
    s, q, lens = batch(cuda, [10], [100], 1, 128, 2)
    clean = fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1).view(-1, 2, 128)
    q[40, 1, 3] = float("nan")
    q[70, 0, 3] = float("inf")
    out = fp8_extend_attention(q, s.pool, s.layer, s.table, *lens, 0.1).view(-1, 2, 128)
    assert out[40, 1].isnan().all() and out[70, 0].isnan().all()
    out[40, 1], out[70, 0] = clean[40, 1], clean[70, 0]
    assert torch.equal(out, clean)


def test_arguments_are_checked(cuda):
    s, q, lens = batch(cuda, [0], [20], 2, 64, 4)

    def call(q=q, table=s.table, lens=lens, scale=0.1):
        return fp8_extend_attention(q, s.pool, s.layer, table, *lens, scale)

    for bad, said in ((dict(q=q.float()), "bfloat16"), (dict(q=q[:, :3]), "divisible"), (dict(q=q.cpu()), "lies on"),
                      (dict(table=s.table.long()), "int32"), (dict(scale=0.0), "positive"), (dict(scale=-1.0), "positive"),
                      (dict(lens=(lens[0], lens[1], lens[2], i64([1, 2], cuda))), "entries"),
                      (dict(lens=tuple(t[:0] for t in lens)), "no request")):
        with pytest.raises(ValueError, match=said):
            call(**bad)
    assert call(q=q[:0]).shape == (0, 256)
    assert torch.equal(call(), call(q=q.view(20, -1), lens=tuple(t.int() for t in lens)))


def test_a_replayed_graph_with_changing_lengths(cuda):
    s, q, _ = batch(cuda, [0, 0], [400, 400], 2, 128, 8)
    rpi, seq, prefix, new = i64([0, 1], cuda), i64([400, 400], cuda), i64([0, 0], cuda), i64([400, 400], cuda)
    args = (q, s.pool, s.layer, s.table, rpi, seq, prefix, new, 0.1)
    fp8_extend_attention(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fp8_extend_attention(*args)
    for a, b, pa, pb in ((400, 400, 0, 0), (1, 300, 99, 64), (390, 0, 10, 0)):
        new.copy_(i64([a, b], cuda))
        prefix.copy_(i64([pa, pb], cuda))
        seq.copy_(new + prefix)
        graph.replay()
        assert torch.equal(out[: a + b], fp8_extend_attention(*args)[: a + b])
        check(s, out[: a + b], q[: a + b], [pa, pb], [a, b], 0.1)
