"""The 4-bit block cache: stores, rows read back and page bounds, equal to the definition."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp4_cache as o4
from qwenquest_amd.paged import Fp4TokenToKVPool
from qwenquest_amd.quest import QuestAlgorithm

pytestmark = pytest.mark.gpu


def i64(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int64).to(dev)


def values(rng, n, kv, dim, dtype):
    """Rows whose sizes, and whose channels' sizes, differ by orders of magnitude."""
    x = rng.standard_normal((n, kv, dim)) * np.exp(2 * rng.standard_normal((1, kv, dim))) * np.exp(3 * rng.standard_normal((n, kv, 1)))
    return torch.from_numpy(x).to(dtype)


def same(pool, cache, layer=0, rows=None):
    rows = np.arange(pool.rows) if rows is None else np.asarray(rows)
    for dtype in (torch.float32, torch.bfloat16):
        for got, want in zip(pool.get_rows(layer, i64(rows, pool.device), dtype), cache.rows(rows)):
            assert got.dtype == dtype
            assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv, dim", [(4, 128), (1, 64), (3, 64), (8, 128), (1, 128)])
def test_rows_written_and_read(cuda, kv, dim, dtype):
    """Runs that begin and end inside blocks, whole blocks, single rows, over and over."""
    rng = np.random.default_rng(kv * dim)
    pool, cache = Fp4TokenToKVPool(64, 2, kv, dim, cuda), o4.Cache(64, kv, dim)
    for lo, hi in ((64, 65), (70, 300), (128, 192), (64, 128), (301, 302), (300, 301), (200, 768), (64, 767), (767, 768), (70, 2500), (2000, 2563), (65, 4095)):
        rows = np.arange(lo, hi)
        k, v = values(rng, len(rows), kv, dim, dtype), values(rng, len(rows), kv, dim, dtype)
        pool.set_kv_buffer(1, i64(rows, cuda), k.to(cuda), v.to(cuda))
        cache.write(rows, k.double().numpy(), v.double().numpy())
        same(pool, cache, 1)
    assert not pool.k_codes[0].any() and (pool.k_scale[0] == 127).all()  # the other layer
    assert not pool.k_codes[1, 0].any() and not pool.v_codes[1, 0].any()  # the padding block


@pytest.mark.parametrize("n", [1, 2, 31, 64, 65, 700, 3900])
def test_scattered_blocks(cuda, n):
    """Entries of many blocks in any order, one and several of a block at a time."""
    rng = np.random.default_rng(n)
    total = 800 if n < 800 else 4000
    pool, cache = Fp4TokenToKVPool(total, 1, 4, 64, cuda), o4.Cache(total, 4, 64)
    for step in range(3):
        blocks = rng.permutation(np.arange(1, total))[:n]
        rows = np.concatenate([b * 64 + rng.permutation(64)[: 1 + (step and rng.integers(0, (5, 64)[step == 2 and n < 800]))] for b in blocks])
        k, v = values(rng, len(rows), 4, 64, torch.bfloat16), values(rng, len(rows), 4, 64, torch.bfloat16)
        pool.set_kv_buffer(0, i64(rows, cuda), k.to(cuda), v.to(cuda))
        cache.write(rows, k.double().numpy(), v.double().numpy())
        same(pool, cache, rows=np.concatenate([np.arange(b * 64, b * 64 + 64) for b in blocks]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv, dim, blocks", [(4, 128, 400), (8, 64, 400), (1, 128, 1200), (3, 64, 800)])
def test_many_entries_at_once(cuda, kv, dim, blocks, dtype):
    """Over a pool, all at once: whole blocks, pieces of them, single rows and rows that are not there, in any order."""
    rng = np.random.default_rng(blocks + dim)
    pool, cache = Fp4TokenToKVPool(blocks, 1, kv, dim, cuda), o4.Cache(blocks, kv, dim)
    for step in range(2):
        pieces = []
        for b in rng.permutation(np.arange(1, blocks)):
            lo, hi = sorted(rng.integers(0, 65, 2)) if rng.random() < 0.3 else (0, 64)
            one = b * 64 + np.arange(lo, hi)
            pieces.append(one if rng.random() < 0.7 else rng.permutation(one)[: rng.integers(1, 65)])
            if rng.random() < 0.1:
                pieces.append(np.array([-1, blocks * 64, 5, 1 << 40]))  # outside the pool, and padding
        rows = np.concatenate(pieces)
        assert len(rows) * kv * dim > 1 << 21
        k, v = values(rng, len(rows), kv, dim, dtype), values(rng, len(rows), kv, dim, dtype)
        pool.set_kv_buffer(0, i64(rows, cuda), k.to(cuda), v.to(cuda))
        cache.write(rows, k.double().numpy(), v.double().numpy())
        everything = np.arange(pool.rows)
        while len(everything) * kv * dim < 7 << 20:
            everything = np.concatenate([everything, everything])
        same(pool, cache, rows=everything)
        same(pool, cache, rows=rng.permutation(everything))
        same(pool, cache, rows=everything[13:-29])
    assert not pool.k_codes[0, 0].any() and not pool.v_codes[0, 0].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_border_and_size(cuda, dtype):
    """Values at and next to the borders between codes, at every exponent, the largest and the least."""
    steps = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.0, 0.5, 1.0, 1.5, 2.0, 3.0], dtype=torch.float64)
    near = torch.cat([steps, steps * (1 + 2.0**-7), steps * (1 - 2.0**-7), -steps])  # 64 channels
    near = near.to(torch.bfloat16).double()
    sizes = torch.arange(-126, 126)
    x = torch.ldexp(near[None].expand(len(sizes), -1), sizes[:, None]).clamp(-3.3e38, 3.3e38)
    x = torch.cat([x[:, None], x.flip(1)[:, None]], 1).to(dtype)  # 2 heads of 64
    flat = x.clone()
    flat[:, :, 10:] = 0  # a token whose second group of K is zeros
    pool, cache = Fp4TokenToKVPool(12, 1, 2, 64, cuda), o4.Cache(12, 2, 64)
    for k, v in ((x, flat), (flat, x)):
        rows = np.arange(64, 64 + len(sizes))
        pool.set_kv_buffer(0, i64(rows, cuda), k.to(cuda), v.to(cuda))
        cache.write(rows, k.double().numpy(), v.double().numpy())
        same(pool, cache)


def test_rows_listed_twice_and_rows_that_are_not_there(cuda):
    rng = np.random.default_rng(3)
    pool, cache = Fp4TokenToKVPool(6, 1, 2, 128, cuda), o4.Cache(6, 2, 128)
    rows = np.array([70, 70, 71, 70, 0, 5, 63, 64 * 6, 64 * 6 + 1, -1, -64, 1 << 40, 130, 131, 130] + [200] * 150 + [201, 200])
    k, v = values(rng, len(rows), 2, 128, torch.bfloat16), values(rng, len(rows), 2, 128, torch.bfloat16)
    pool.set_kv_buffer(0, i64(rows, cuda), k.to(cuda), v.to(cuda))
    cache.write(rows, k.double().numpy(), v.double().numpy())
    same(pool, cache)
    got = pool.get_rows(0, i64([70, -1, 384, 1 << 40, 0], cuda))
    for x in got:
        assert x[1:4].isnan().all() and not x[[0, 4]].isnan().any()
    pool.set_kv_buffer(0, i64([], cuda), k[:0].to(cuda), v[:0].to(cuda))
    assert pool.get_rows(0, i64([], cuda))[0].shape == (0, 2, 128)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_not_finite_is_lost_alone(cuda, dtype, dim):
    """A (token, head) with a NaN, an infinity or a V too large reads NaN, its neighbours as ever; written
    again it is whole."""
    rng = np.random.default_rng(1)
    pool, cache = Fp4TokenToKVPool(4, 1, 3, dim, cuda), o4.Cache(4, 3, dim)
    rows = np.arange(64, 256)
    k, v = values(rng, 192, 3, dim, dtype), values(rng, 192, 3, dim, dtype)
    for i, (t, h, d, x, bad) in enumerate(((0, 0, 0, k, "nan"), (17, 1, dim - 1, v, "inf"), (33, 2, 40, k, "-inf"), (64, 0, 5, v, "nan"),
                                           (100, 1, 33, v, str(7.25 * 2.0**59)), (101, 1, 33, v, str(7 * 2.0**59)), (191, 2, 63, v, "-3e38"))):
        x[t, h, d] = float(bad)
    pool.set_kv_buffer(0, i64(rows, cuda), k.to(cuda), v.to(cuda))
    cache.write(rows, k.double().numpy(), v.double().numpy())
    assert np.isnan(cache.rows(rows)[0]).any(-1).sum() == 6 and not np.isnan(cache.rows([64 + 101])[1]).any()
    same(pool, cache)
    for t in (0, 17, 191):  # one at a time, as a decode step writes
        k, v = values(rng, 1, 3, dim, dtype), values(rng, 1, 3, dim, dtype)
        pool.set_kv_buffer(0, i64([64 + t], cuda), k.to(cuda), v.to(cuda))
        cache.write([64 + t], k.double().numpy(), v.double().numpy())
    same(pool, cache)


def test_strided_and_unaligned_rows_and_other_types(cuda):
    pool, cache = Fp4TokenToKVPool(4, 1, 2, 64, cuda), o4.Cache(4, 2, 64)
    base = torch.randn(20, 4, 64, device=cuda)
    odd = torch.randn(10 * 2 * 64 + 1, device=cuda)[1:].view(10, 2, 64)
    for k, v in ((base[::2, :2], base[1::2, 2:]), (odd, odd * 3), (odd.half(), odd.half() * 2), (odd.double(), base[::2, :2])):
        rows = np.arange(64, 74)
        pool.set_kv_buffer(0, i64(rows, cuda).int(), k, v)
        cache.write(rows, k.float().double().cpu().numpy(), v.float().double().cpu().numpy())
        same(pool, cache)


def test_a_large_pool(cuda):
    """Blocks whose codes lie past 2^32 bytes."""
    blocks = 70000
    pool = Fp4TokenToKVPool(blocks, 1, 16, 128, cuda)
    assert pool.k_codes.numel() > 1 << 32
    rng = np.random.default_rng(0)
    rows = np.concatenate([np.arange(b * 64, b * 64 + 64) for b in (1, blocks // 2, blocks - 1)])
    k, v = values(rng, len(rows), 16, 128, torch.bfloat16), values(rng, len(rows), 16, 128, torch.bfloat16)
    cache = o4.Cache(4, 16, 128)
    cache.write(np.arange(64, 256), k.double().numpy(), v.double().numpy())
    pool.set_kv_buffer(0, i64(rows, cuda), k.to(cuda), v.to(cuda))
    for got, want in zip(pool.get_rows(0, i64(rows, cuda)), cache.rows(np.arange(64, 256))):
        assert np.array_equal(got.double().cpu().numpy(), want)


@pytest.mark.parametrize("n", [10, 500])
def test_on_another_stream_and_captured(cuda, n):
    pool, cache = Fp4TokenToKVPool(20, 1, 2, 128, cuda), o4.Cache(20, 2, 128)
    rng = np.random.default_rng(n)
    rows = np.arange(70, 70 + n)
    loc, k, v = i64(rows, cuda), *(torch.zeros(n, 2, 128, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pool.set_kv_buffer(0, loc, k, v)
        pool.get_rows(0, loc)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.set_kv_buffer(0, loc, k, v)
        got = pool.get_rows(0, loc)
    for _ in range(3):
        kn, vn = values(rng, n, 2, 128, torch.bfloat16), values(rng, n, 2, 128, torch.bfloat16)
        k.copy_(kn)
        v.copy_(vn)
        graph.replay()
        cache.write(rows, kn.double().numpy(), vn.double().numpy())
        for x, want in zip(got, cache.rows(rows)):
            assert np.array_equal(x.double().cpu().numpy(), want)
        torch.zeros(1000, device=cuda).sum().item()


def test_arguments_are_checked(cuda):
    pool = Fp4TokenToKVPool(4, 2, 2, 64, cuda)
    x = torch.zeros(3, 2, 64, device=cuda)
    loc = i64([64, 65, 66], cuda)
    for args, said in (((0, loc, x[:2], x), "rows"), ((0, loc, x, x.view(3, 4, 32)[:, :3]), "rows"), ((0, loc.view(1, 3), x, x), "one-dim"),
                       ((0, loc.float(), x, x), "whole numbers")):
        with pytest.raises(ValueError, match=said):
            pool.set_kv_buffer(*args)
    with pytest.raises(IndexError):
        pool.set_kv_buffer(2, loc, x, x)
    with pytest.raises(RuntimeError, match="GPU"):
        pool.set_kv_buffer(0, loc, x.cpu(), x.cpu())
    with pytest.raises(ValueError, match="dtype"):
        pool.get_rows(0, loc, torch.float16)
    for bad in (dict(head_dim=96), dict(head_dim=256), dict(num_blocks=0), dict(kv_heads=0), dict(num_layers=0)):
        with pytest.raises(ValueError):
            Fp4TokenToKVPool(**{**dict(num_blocks=4, num_layers=1, kv_heads=1, head_dim=64, device=cuda), **bad})
    assert pool.storage_bytes() == 2 * 4 * 2 * (64 * 64 + 2 * 64 + 64)


# ---------------------------------------------------------------- page bounds


def bits(x: np.ndarray) -> np.ndarray:
    return torch.from_numpy(x).to(torch.bfloat16).double().numpy()


@pytest.mark.parametrize("kv, dim", [(4, 128), (3, 64), (8, 128)])
@pytest.mark.parametrize("decode", [False, True])
def test_page_bounds(cuda, kv, dim, decode):
    """Of the pages that are complete (decode: by the token before the step's), at every Quest layer; a page
    with a lost token, and one whose block is not there, NaN."""
    rng = np.random.default_rng(kv + dim)
    lens = [64, 65, 63, 300, 0, 1, 257, 128 + 1]
    blocks, layers = 40, 3
    pool = Fp4TokenToKVPool(blocks, layers, kv, dim, cuda)
    caches = [o4.Cache(blocks, kv, dim) for _ in range(layers)]
    rows = np.arange(64, blocks * 64)
    for layer in range(layers):
        k, v = values(rng, len(rows), kv, dim, torch.bfloat16), values(rng, len(rows), kv, dim, torch.bfloat16)
        k[130, kv - 1, 3] = float("nan")
        pool.set_kv_buffer(layer, i64(rows, cuda), k.to(cuda), v.to(cuda))
        caches[layer].write(rows, k.double().numpy(), v.double().numpy())
    ids = (1 + rng.permutation(blocks - 1)).tolist()
    table = np.zeros((len(lens), 6), dtype=np.int32)
    for r, n in enumerate(lens):
        for j in range(-(-n // 64)):
            table[r, j] = ids.pop()
    table[3, 1] = blocks  # outside the pool
    q = QuestAlgorithm(128, 64, cuda)
    q.init_storage(1, layers, len(lens), 6 * 64, kv, dim)
    before = q.page_k_bounds.clone()
    reqs = [3, 0, 1, 2, 7, 6, 5, 4]
    seq = i64([lens[r] for r in reqs], cuda)
    t = torch.from_numpy(table).to(cuda)
    if decode:
        step = q.decode_step_blocks(i64(reqs, cuda), seq, pool, t)
        assert step.actual_lens.tolist() == [min(lens[r], 128) for r in reqs]
        assert step.candidate_limit_i32.tolist() == [max(lens[r] - 1, 0) // 64 for r in reqs]
    else:
        q.update_prefill_representations_blocks(i64(reqs, cuda), seq, pool, t)
    got = q.page_k_bounds.double().cpu().numpy()
    want = before.double().cpu().numpy()
    for li, layer in enumerate(range(1, layers)):
        for r, n in enumerate(lens):
            pages = ([(n - 1) // 64 - 1] if n >= 2 and (n - 1) % 64 == 0 else []) if decode else range(n // 64)
            for p in pages:
                if table[r, p] >= blocks:
                    want[li, r, p] = np.nan
                    continue
                k = caches[layer].rows(np.arange(table[r, p] * 64, table[r, p] * 64 + 64))[0]
                lost = np.isnan(k).any(0)
                with np.errstate(invalid="ignore"):
                    pair = np.stack([bits(k.min(0)), bits(k.max(0))], -1)
                want[li, r, p] = np.where(lost.any(-1)[:, None, None], np.nan, pair)
    assert np.array_equal(got.reshape(want.shape), want, equal_nan=True)
