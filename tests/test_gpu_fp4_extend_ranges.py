"""Prefill over the 4-bit block cache at the ends of what the cache holds: values at both ends of V's range, bytes
behind a context that nobody wrote, scores far past 2^24.  References and tolerances: tests/test_gpu_fp4_extend.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_fp4_extend import batch, check, run

pytestmark = pytest.mark.gpu


def two_kinds(cuda, prefix, new, dim, heads, gap, at, low):
    """One token (position `at`) of values near 7 * 2^59 that weighs 2^gap of each other one, whose values are `low` in size."""
    s, q, lens = batch(cuda, [prefix], [new], 1, dim, heads, seed=dim)
    n = prefix + new
    gen = torch.Generator(device=cuda).manual_seed(n)
    k = torch.empty((n, 1, dim), device=cuda).normal_(generator=gen) * 2.0**-6
    v = torch.empty((n, 1, dim), device=cuda).normal_(generator=gen).clamp_(-6, 6) * low
    one = torch.empty(dim, device=cuda).uniform_(2.0, 6.5, generator=gen)
    k[..., 0] = -4.0
    k[at, 0, 0] = 4.0
    v[at, 0] = one * torch.where(torch.arange(dim, device=cuda) % 3 == 0, -1.0, 1.0) * 2.0**59
    s.pool.set_kv_buffer(s.layer, s.rows(0, np.arange(n)), k, v)
    q.mul_(2.0**-6)
    q[..., 0] = gap / 8 * 0.6931  # at a scale of 1: 2^gap between the two
    return s, q, lens


@pytest.mark.parametrize("low", [2.0**-51, 0.0])
@pytest.mark.parametrize("gap", [17.0, 18.5, 20.0])
@pytest.mark.parametrize("prefix, new, heads, dim", [(8192, 600, 32, 64), (8192, 300, 64, 128), (8192, 3, 4, 128), (20000, 5, 2, 64)])
def test_the_sum_over_the_whole_range_of_values(cuda, prefix, new, heads, dim, gap, low):
    """Thousands of tokens at the low end of V's range before one at its high end: whole query tiles and splits.  In the
    weights' sum all of them count: 8192 times 2^-17 is a sixteenth of it."""
    s, q, lens = two_kinds(cuda, prefix, new, dim, heads, gap, prefix - 1, low)
    check(s, run(s, q, lens, 1.0), q, [prefix], [new], 1.0)


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("new, heads", [(3, 2), (280, 64)])
def test_the_sum_where_weights_of_the_products_underflow(cuda, new, heads, first):
    """2^18 tokens without values that weigh 2^-24.5 of one with the largest: 2^(-24.5 - 50 - 59 + 7) is no normal float32,
    and still they are a ninetieth of the sum.  All terms are positive: what sums in float32 lose is, of each
    term, half a step for each of a chain of 32 in a tile, one for each tile, and those of the splits."""
    prefix, gap = (1 << 18), 24.5
    s, q, lens = two_kinds(cuda, prefix, new, 64, heads, gap, 0 if first else prefix - 1, 0.0)
    out = run(s, q, lens, 1.0).double().view(q.shape)
    n = prefix + new
    k, v = (x.double()[:, 0] for x in s.pool.get_rows(s.layer, s.rows(0, np.arange(n)), torch.float32))
    pick = list(range(0, new, 93)) + [new - 1]
    qh = q[pick].double()
    t = (qh.reshape(-1, 64) @ k.T.contiguous()).view(len(pick), heads, n)
    seen = torch.arange(n, device=cuda)[None] <= prefix + torch.tensor(pick, device=cuda)[:, None]
    w = torch.softmax(t.masked_fill(~seen[:, None], -np.inf), -1)
    want, spread = (w.view(-1, n) @ v).view(out[pick].shape), (w.view(-1, n) @ v.abs()).view(out[pick].shape)
    size = (qh.abs().reshape(-1, 64) @ k.abs().T.contiguous()).amax(-1).view(len(pick), heads, 1)
    tol = 2.0**-8 * want.abs() + (2.0**-10 + 2 * 68 * 2.0**-23 * size + (32 + n / 64 + 32) * 2.0**-24) * spread
    assert float(1 - w.amax(-1).max()) > 0.008
    err = (out[pick] - want).abs()
    assert (err <= tol).all(), f"off by {(err / tol).max().item():.2f} tolerances"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix, new, heads", [([0, 63, 100], [1, 70, 130], 4), ([3000], [7], 2), ([700], [600], 64)])
def test_bytes_that_nobody_wrote(cuda, prefix, new, heads, dim):
    """Whatever the cache's bytes are behind a context, in the block in which it ends: the same answers, to the bit."""
    s, q, lens = batch(cuda, prefix, new, 1, dim, heads, seed=dim)
    kept = [s.pool.get_rows(s.layer, s.rows(i, np.arange(n)), torch.float32) for i, n in enumerate(s.lens)]
    ref = run(s, q, lens, 0.1)
    check(s, ref, q, prefix, new, 0.1)
    for codes, scale in ((0, 0), (0x77, 0), (0xFF, 255), (0x91, 254), (0x2F, 1), (0x77, 200)):
        for t in (s.pool.k_codes, s.pool.v_codes):
            t.fill_(codes)
        for t in (s.pool.k_scale, s.pool.v_scale):
            t.fill_(scale)
        for i, (k, v) in enumerate(kept):  # exact: the cache's own values
            s.pool.set_kv_buffer(s.layer, s.rows(i, np.arange(s.lens[i])), k, v)
        assert torch.equal(run(s, q, lens, 0.1), ref), (codes, scale)


@pytest.mark.parametrize("dim, prefix, new, pad_heads", [(64, 0, 120, 2), (128, 0, 120, 2), (64, 90, 30, 2), (128, 117, 3, 64)])
def test_scores_far_past_2_24(cuda, dim, prefix, new, pad_heads):
    """Scores that grow from 2^7 to 2^66 (and fall to -2^66 for the other sign): a row's output is the value of its largest
    score, every other one being a power of two of e below it."""
    n = prefix + new
    s, q, lens = batch(cuda, [prefix], [new], 1, dim, pad_heads, seed=1)
    j = torch.arange(n, device=cuda)
    k = torch.zeros((n, 1, dim), device=cuda)
    k[:, 0, 0] = (1 + (j % 2) / 2) * torch.exp2((7 + j // 2).float())
    v = torch.randn((n, 1, dim), device=cuda)
    s.pool.set_kv_buffer(s.layer, s.rows(0, np.arange(n)), k, v)
    q.zero_()
    q[:, 0::2, 0], q[:, 1::2, 0] = 1.0, -1.0
    out = run(s, q, lens, 1.0).view(new, pad_heads, dim)
    vals = s.pool.get_rows(s.layer, s.rows(0, np.arange(n)), torch.bfloat16)[1][:, 0]
    assert torch.equal(out[:, 0::2], vals[prefix:][:, None].expand(-1, pad_heads // 2, -1))
    assert torch.equal(out[:, 1::2], vals[:1][:, None].expand(new, pad_heads // 2, -1))


@pytest.mark.parametrize("exponent", [10, 23, 24, 26, 27, 28, 33, 60, 100])
def test_equal_scores_of_any_size_weigh_the_same(cuda, exponent):
    """A mean over the context, whatever the score that all tokens share.  Weights alike, their common rounding (2^-10 at
    most) cancels against the sum's but for what truncation keeps of it; half a step of bf16."""
    s, q, lens = batch(cuda, [70], [30], 1, 64, 4, seed=2)
    k, v = torch.zeros((100, 1, 64), device=cuda), torch.randn((100, 1, 64), device=cuda)
    k[..., 0] = 1.5 * 2.0**exponent
    v[..., 0] = 6.0  # one scale for all
    s.pool.set_kv_buffer(s.layer, s.rows(0, np.arange(100)), k, v.clamp_(-6, 6))
    q.zero_()
    q[:, :2, 0], q[:, 2:, 0] = 1.0, -1.0
    out = run(s, q, lens, 1.0).view(30, 4, 64).double()
    vals = s.pool.get_rows(s.layer, s.rows(0, np.arange(100)), torch.float32)[1][:, 0].double()
    for t in range(30):
        want, spread = vals[: 71 + t].mean(0), vals[: 71 + t].abs().mean(0)
        assert ((out[t] - want).abs() <= 2.0**-8 * want.abs() + (2.0**-10 + 100 * 2.0**-23) * spread).all(), t
