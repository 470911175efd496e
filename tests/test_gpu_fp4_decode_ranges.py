"""Decode over the 4-bit block cache with scores far past 2^24, and with bytes behind a context that nobody wrote."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qwenquest_amd.attention.ops import fp4_decode_attention, fp4_decode_plan
from tests.test_gpu_fp4_decode import Setup, i64, picked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim, heads, kv", [(128, 4, 2), (64, 34, 1)])
@pytest.mark.parametrize("scale", [1.0, -1.0])
def test_scores_far_past_2_24(cuda, dim, heads, kv, dtype, scale):
    """Scores that grow from 2^7 to 2^66 (and fall to -2^66 for the other sign): the output is the mean value of those that
    share the largest.  Every other one is 64 at least below it: 120 tokens of e^-64 < 2^-92 and values under 2^4 are
    less than 2^-80.  A mean of two values of 2 bits each, by a sum of two weights: two roundings of float32, and bf16's."""
    s = Setup(cuda, [120, 64 * 40], kv, dim, seed=1)
    values = []
    for r, n in enumerate(s.lens):
        j = torch.arange(n, device=cuda)
        k = torch.zeros((n, kv, dim), device=cuda)
        k[:, :, 0] = ((1 + (j % 2) / 2) * torch.exp2((7 + (j // 2) * 60 // n * 2).float()))[:, None] if r == 0 else 2.0**40
        if r == 1:
            k[1717, :, 0] = 1.5 * 2.0**40
        s.pool.set_kv_buffer(s.layer, s.rows(r, np.arange(n)), k, torch.randn((n, kv, dim), device=cuda))
        values.append(s.pool.get_rows(s.layer, s.rows(r, np.arange(n)), torch.float32)[1])
    lens = [1, 2, 3, 33, 64, 65, 100, 120]
    q = torch.zeros((len(lens) + 1, heads, dim), device=cuda, dtype=dtype)
    q[..., 0] = 1.0
    q[:-1, 1::2, 0] = -1.0
    reqs, n = i64([0] * len(lens) + [1], cuda), i64([*lens, s.lens[1]], cuda)
    k0 = s.pool.get_rows(s.layer, s.rows(0, np.arange(120)), torch.float32)[0][:, 0, 0]
    for plan in (None, fp4_decode_plan(s.pool, s.table, reqs, n)):
        out = fp4_decode_attention(q, s.pool, s.layer, s.table, reqs, n, scale, plan=plan).view(-1, heads, dim).float()
        for i, m in enumerate([*lens, 0]):
            for h in range(heads):
                sign = scale * (1.0 if h % 2 == 0 else -1.0)
                if m == 0 and scale < 0:
                    continue  # 2559 equal ones and one below
                t = k0[:m] * sign
                at = [1717] if m == 0 else (t == t.max()).nonzero()[:, 0]
                v = values[1 if m == 0 else 0][at, h * kv // heads].double()
                want, half = v.mean(0), 2.0**-8 if dtype == torch.bfloat16 else 2.0**-24
                assert ((out[i, h] - want).abs() <= half * want.abs() + 2.0**-22 * v.abs().mean(0) + 2.0**-80).all(), (m, h)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("exponent", [10, 24, 28, 31, 33, 36, 60, 100])
def test_equal_scores_of_any_size_weigh_the_same(cuda, exponent, dtype):
    """A mean over the context, whatever the score that all tokens share: sums of n terms in float32."""
    n = 777
    s = Setup(cuda, [n], 1, 64, seed=2)
    k, v = torch.zeros((n, 1, 64), device=cuda), torch.randn((n, 1, 64), device=cuda)
    k[..., 0] = 1.5 * 2.0**exponent
    s.pool.set_kv_buffer(s.layer, s.rows(0, np.arange(n)), k, v)
    v = s.pool.get_rows(s.layer, s.rows(0, np.arange(n)), torch.float32)[1][:, 0].double()
    q = torch.zeros((1, 4, 64), device=cuda, dtype=dtype)
    q[:, :2, 0], q[:, 2:, 0] = 1.0, -1.0
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, i64([0], cuda), i64([n], cuda), 1.0).view(4, 64).double()
    half = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-24
    assert ((out - v.mean(0)).abs() <= half * v.mean(0).abs() + n * 2.0**-23 * v.abs().mean(0)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
def test_bytes_that_nobody_wrote(cuda, dim, dtype):
    """Whatever the cache's bytes are behind a context, in the blocks in which it ends: the same answers, to the bit,
    of whole contexts and of a selection with its window."""
    lens = [1, 63, 64, 100, 130, 700]
    s = Setup(cuda, lens, 2, dim, seed=4)
    q, reqs, n = s.queries(8, dtype), torch.arange(len(lens), device=cuda), i64(lens, cuda)
    kept = [s.pool.get_rows(s.layer, s.rows(i, np.arange(m)), torch.float32) for i, m in enumerate(lens)]
    pos = np.zeros((len(lens), 128), dtype=np.int32)
    pos[5], pos[4] = picked(None, 700, 128, pages=[3]), picked(None, 130, 128, pages=[0])
    pos = torch.from_numpy(pos).to(cuda)

    def both():
        args = (q, s.pool, s.layer, s.table, reqs, n, 0.1)
        return fp4_decode_attention(*args), fp4_decode_attention(*args, positions=pos, top_k=128)

    ref = both()
    s.check(ref[0], q, 0.1)
    for codes, scale in ((0, 0), (0x77, 0), (0xFF, 255), (0x91, 254), (0x2F, 1), (0x77, 200)):
        for t in (s.pool.k_codes, s.pool.v_codes):
            t.fill_(codes)
        for t in (s.pool.k_scale, s.pool.v_scale):
            t.fill_(scale)
        for i, (k, v) in enumerate(kept):
            s.pool.set_kv_buffer(s.layer, s.rows(i, np.arange(lens[i])), k, v)
        assert all(torch.equal(a, b) for a, b in zip(both(), ref)), (codes, scale)
