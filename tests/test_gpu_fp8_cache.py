"""The 8-bit block cache: stores, rows read back and page bounds, equal to the definition bit for bit."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from oracle import fp8_cache as of
from qwenquest_amd.paged import Fp8TokenToKVPool
from qwenquest_amd.quest import QuestAlgorithm

pytestmark = pytest.mark.gpu

FAR = torch.finfo(torch.bfloat16).max


def i64(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int64).to(dev)


def same(a, b):
    return np.array_equal(np.asarray(a, dtype=np.float64), np.asarray(b, dtype=np.float64), equal_nan=True)


def check(pool, want, layer=0):
    """Every row of every block but the padding one, and every scale."""
    loc = torch.arange(64, pool.rows)
    for dtype in (torch.bfloat16, torch.float32):
        k, v = pool.get_rows(layer, loc, dtype)
        # as float32: 3.3e38 / 2^120 = 248.3 rounds to the code 256, and 256 * 2^120 = 2^128 is infinite
        with np.errstate(over="ignore"):
            wk, wv = (x.astype(np.float32) for x in want.rows(loc.numpy()))
        assert same(k.float().cpu().numpy(), wk) and same(v.float().cpu().numpy(), wv)
    assert same(pool.k_scale[layer].cpu().numpy(), want.scale(0)) and same(pool.v_scale[layer].cpu().numpy(), want.scale(1))


def values(rng, n, kv, dim, spread=3.0):
    """Magnitudes over many binary orders, a few zeros."""
    x = rng.standard_normal((n, kv, dim)) * np.exp2(rng.normal(0, spread, (n, kv, 1)))
    x[rng.random(x.shape) < 0.05] = 0.0
    return x.astype(np.float32)


@pytest.mark.parametrize("kv, dim, dtype", [(1, 128, torch.bfloat16), (4, 128, torch.float32), (3, 64, torch.bfloat16),
                                            (8, 64, torch.float32), (5, 128, torch.bfloat16)])
def test_runs_of_every_kind(cuda, kv, dim, dtype):
    """Whole blocks, parts of blocks begun and gone on with, single tokens, growth of the scale."""
    rng = np.random.default_rng(kv * dim)
    blocks = 12
    pool, want = Fp8TokenToKVPool(blocks, 2, kv, dim, cuda), of.Cache(blocks, kv, dim)
    runs = [[*range(64, 64 + 200)], [*range(64 + 200, 64 + 256), *range(64 * 7, 64 * 7 + 1)], [*range(64 * 7 + 1, 64 * 7 + 64)],
            [64 * 9 + i for i in range(30)], [64 * 9 + 30], [64 * 9 + 31, 64 * 10], [64 * 9 + 33, 64 * 10 + 5, 64 * 7 + 3],
            [64 * 3], [64 * 9, 64 * 9 + 1]]
    for i, loc in enumerate(runs):
        k, v = (torch.from_numpy(values(rng, len(loc), kv, dim)).to(cuda, dtype) for _ in range(2))
        if i == 4:
            k *= 1000.0  # the scale grows in one head's direction or all
            v *= 30000.0
        pool.set_kv_buffer(1, i64(loc, cuda), k, v)
        want.write(loc, k.float().cpu().numpy(), v.float().cpu().numpy())
        check(pool, want, 1)
    assert not pool.k_codes[0].any() and not pool.k_codes[1, 0].any()


@pytest.mark.parametrize("seed", range(3))
def test_a_decode_life(cuda, seed):
    """Requests that grow token by token, each in its own blocks, in batches with padding."""
    rng = np.random.default_rng(seed)
    kv, dim, bs, blocks = 2, 128, 9, 40
    pool, want = Fp8TokenToKVPool(blocks, 1, kv, dim, cuda), of.Cache(blocks, kv, dim)
    lens = rng.integers(0, 70, bs)
    for step in range(75):
        loc = [64 * (1 + 4 * b) + int(lens[b]) if rng.random() < 0.9 else 0 for b in range(bs)]
        k, v = (torch.from_numpy(values(rng, bs, kv, dim)).to(cuda, torch.bfloat16) for _ in range(2))
        pool.set_kv_buffer(0, i64(loc, cuda), k, v)
        want.write(loc, k.float().cpu().numpy(), v.float().cpu().numpy())
        for b in range(bs):
            lens[b] += loc[b] > 0
        if step % 25 == 24:
            check(pool, want)


def test_a_prompt_longer_than_one_round(cuda):
    """More entries than the store looks at one by one, its runs beginning anywhere in a segment."""
    rng = np.random.default_rng(1)
    kv, dim, blocks = 2, 64, 120
    pool, want = Fp8TokenToKVPool(blocks, 1, kv, dim, cuda), of.Cache(blocks, kv, dim)
    order = rng.permutation(np.arange(1, blocks))
    loc = np.concatenate([b * 64 + np.arange(rng.choice([1, 17, 63, 64, 64, 64])) for b in order])
    assert len(loc) > 4096
    k, v = (torch.from_numpy(values(rng, len(loc), kv, dim)).to(cuda) for _ in range(2))
    pool.set_kv_buffer(0, i64(loc, cuda), k, v)
    want.write(loc, k.cpu().numpy(), v.cpu().numpy())
    check(pool, want)


@pytest.mark.parametrize("n, kv", [(600, 2), (600, 5), (1500, 2), (1500, 6), (1500, 11), (1025, 1), (1024, 1)])
def test_segments_of_every_length(cuda, n, kv):
    """2 to 64 entries looked after together: runs of a block's whole length and of single entries."""
    rng = np.random.default_rng(n * kv)
    dim, blocks = 64, 260
    pool, want = Fp8TokenToKVPool(blocks, 1, kv, dim, cuda), of.Cache(blocks, kv, dim)
    loc = []
    for b in rng.permutation(np.arange(1, blocks)):
        first, many = int(rng.integers(0, 64)), int(rng.choice([1, 1, 2, 30, 64, 64]))
        loc += [int(b) * 64 + t for t in range(first, min(first + many, 64))] + [0] * int(rng.random() < 0.1)
    while len(loc) < n:
        loc.append(loc[-1])  # the last row, over and over
    loc = np.array(loc[-n:])
    for _ in range(2):
        k, v = (torch.from_numpy(values(rng, n, kv, dim)).to(cuda) for _ in range(2))
        pool.set_kv_buffer(0, i64(loc, cuda), k, v)
        want.write(loc, k.cpu().numpy(), v.cpu().numpy())
        check(pool, want)


def test_edges_of_the_format(cuda):
    """Ties, subnormal codes, the largest code, the least scale, zeros, signs."""
    kv, dim = 1, 64
    pool, want = Fp8TokenToKVPool(9, 1, kv, dim, cuda), of.Cache(9, kv, dim)
    rows = {64: np.linspace(-448, 448, dim), 128: 448 * np.exp2(-np.arange(dim, dtype=np.float64)),
            192: np.arange(dim) * 2.0**-11, 256: np.full(dim, 1e-38), 320: np.full(dim, 3.3e38),
            384: np.concatenate([np.zeros(dim - 1), [448.00003]]), 448: np.zeros(dim), 449: -np.full(dim, 2.0**-100)}
    rows[193] = np.full(dim, 448.0)  # raises the scale over codes that turn subnormal
    rows[194] = np.full(dim, 448.0 * 2**9)
    for loc, x in rows.items():
        x = x.astype(np.float32).reshape(1, kv, dim)
        pool.set_kv_buffer(0, i64([loc], cuda), torch.from_numpy(x).to(cuda), torch.from_numpy(-x).to(cuda))
        want.write([loc], x, -x)
        check(pool, want)


@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite(cuda, poison):
    """They spoil their (block, head), K and V apart, until the block is begun again."""
    rng = np.random.default_rng(5)
    kv, dim = 3, 64
    pool, want = Fp8TokenToKVPool(4, 1, kv, dim, cuda), of.Cache(4, kv, dim)
    for loc, bad in ((range(64, 90), False), (range(90, 92), True), (range(92, 100), False), (range(128, 192), False),
                     (range(64, 65), False)):
        loc = [*loc]
        k, v = values(rng, len(loc), kv, dim), values(rng, len(loc), kv, dim)
        if bad:
            k[1, 1, 7] = poison
            v[0, 2, 63] = poison
        pool.set_kv_buffer(0, i64(loc, cuda), *(torch.from_numpy(x).to(cuda) for x in (k, v)))
        want.write(loc, k, v)
        check(pool, want)
    assert (pool.k_codes & 0x7F != 0x7F).all() and (pool.v_codes & 0x7F != 0x7F).all()  # no NaN among the codes


def test_rows_that_are_skipped_and_listed_twice(cuda):
    rng = np.random.default_rng(3)
    kv, dim = 2, 128
    pool, want = Fp8TokenToKVPool(5, 1, kv, dim, cuda), of.Cache(5, kv, dim)
    loc = [0, 63, 64, 65, 65, 64, 70, -1, -(1 << 62), 64 * 5, 1 << 62, 128, 128, 128, 5]
    k, v = (torch.from_numpy(values(rng, len(loc), kv, dim)).to(cuda) for _ in range(2))
    pool.set_kv_buffer(0, i64(loc, cuda), k, v)
    want.write(loc, k.cpu().numpy(), v.cpu().numpy())
    check(pool, want)
    assert not pool.k_codes[0, 0].any()
    k, v = pool.get_rows(0, i64([-1, 64 * 5, 1 << 60, 64, 0], cuda))
    assert k[:3].isnan().all() and v[:3].isnan().all() and not k[3:].isnan().any() and not k[4].any()
    # a run longer than a block, by repetition
    loc = [192] * 150 + [193] * 3
    k, v = (torch.from_numpy(values(rng, len(loc), kv, dim)).to(cuda) for _ in range(2))
    pool.set_kv_buffer(0, i64(loc, cuda), k, v)
    want.write(loc, k.cpu().numpy(), v.cpu().numpy())
    check(pool, want)


def test_layouts_types_and_refusals(cuda):
    rng = np.random.default_rng(4)
    kv, dim = 2, 64
    pool, want = Fp8TokenToKVPool(4, 1, kv, dim, cuda), of.Cache(4, kv, dim)
    n = 70
    base = torch.from_numpy(values(rng, n, 2 * kv, dim)).to(cuda)
    loc = torch.arange(64, 64 + n, dtype=torch.int32, device=cuda)
    kv_pair = base.view(n, 2, kv, dim)
    pool.set_kv_buffer(0, loc, kv_pair[:, 0], kv_pair[:, 1].double())  # strided views, int32 rows, mixed types
    want.write(loc.cpu().numpy(), *(kv_pair[:, i].cpu().numpy() for i in range(2)))
    check(pool, want)
    flat = torch.empty(n * kv * dim + 1, device=cuda)[1:]  # 4 bytes past an aligned address
    flat.copy_(base[:, :kv].reshape(-1))
    pool.set_kv_buffer(0, loc, flat.view(n, kv * dim), flat.view(n, kv * dim).to(torch.float16))
    x = flat.view(n, kv, dim)
    want.write(loc.cpu().numpy(), x.cpu().numpy(), x.half().float().cpu().numpy())
    check(pool, want)
    pool.set_kv_buffer(0, loc[:0], x[:0], x[:0])
    assert pool.get_rows(0, loc[:0])[0].shape == (0, kv, dim)
    with pytest.raises(ValueError, match="rows"):
        pool.set_kv_buffer(0, loc, x[:5], x)
    with pytest.raises(IndexError):
        pool.set_kv_buffer(1, loc, x, x)
    with pytest.raises(ValueError, match="dtype"):
        pool.get_rows(0, loc, torch.float16)
    with pytest.raises(ValueError, match="whole"):
        pool.get_rows(0, loc.float())
    for bad in (dict(head_dim=96), dict(kv_heads=0), dict(num_layers=0), dict(num_blocks=0)):
        with pytest.raises(ValueError):
            Fp8TokenToKVPool(**{**dict(num_blocks=3, num_layers=1, kv_heads=2, head_dim=64, device=cuda), **bad})


def test_a_store_in_a_replayed_graph_and_on_another_stream(cuda):
    rng = np.random.default_rng(6)
    kv, dim = 2, 128
    pool, want = Fp8TokenToKVPool(6, 1, kv, dim, cuda), of.Cache(6, kv, dim)
    loc = i64([64, 128], cuda)
    k, v = (torch.zeros(2, kv, dim, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pool.set_kv_buffer(0, loc, k, v)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            pool.set_kv_buffer(0, loc, k, v)
    torch.cuda.synchronize()
    for _ in range(5):
        for t in (k, v):
            t.copy_(torch.from_numpy(values(rng, 2, kv, dim)))
        graph.replay()
        want.write(loc.cpu().numpy(), k.float().cpu().numpy(), v.float().cpu().numpy())
        check(pool, want)
        loc += 1


# ---------------------------------------------------------------- page bounds


def table_of(blocks, dev, cols):
    t = torch.zeros((len(blocks), cols), dtype=torch.int32, device=dev)
    for r, b in enumerate(blocks):
        t[r, : len(b)] = torch.tensor(b, dtype=torch.int32)
    return t


@pytest.mark.parametrize("kv, dim, layers", [(1, 64, 3), (4, 128, 2), (5, 128, 1), (2, 64, 1)])
def test_bounds_of_prompts_and_of_decode_steps(cuda, kv, dim, layers):
    rng = np.random.default_rng(kv + dim)
    lens = [0, 63, 64, 500, 129]
    ids = (1 + np.random.default_rng(0).permutation(40)).tolist()
    blocks = []
    for n in lens:
        blocks.append([ids.pop() for _ in range(-(-(n + 70) // 64))])
    pool = Fp8TokenToKVPool(41, layers + 1, kv, dim, cuda)
    want = [of.Cache(41, kv, dim) for _ in range(layers + 1)]
    table = table_of(blocks, cuda, 12)
    quest = QuestAlgorithm(128, 64, cuda)
    quest.init_storage(1, layers + 1, len(lens), 12 * 64, kv, dim)  # the Quest layers start at model layer 1

    def write(layer, loc):
        k, v = (values(rng, len(loc), kv, dim) for _ in range(2))
        pool.set_kv_buffer(layer, i64(loc, cuda), torch.from_numpy(k).to(cuda), torch.from_numpy(v).to(cuda))
        want[layer].write(loc, k, v)

    def rows(r, lo, hi):
        return [blocks[r][p // 64] * 64 + p % 64 for p in range(lo, hi)]

    def expect(full):
        got = quest.page_k_bounds.float().cpu().numpy()
        for layer in range(1, layers + 1):
            for r in range(len(lens)):
                k = want[layer].values[0][blocks[r]]
                for p in range(12):
                    lo, hi = (k[p].min(0), k[p].max(0)) if p < full[r] else (FAR, -FAR)
                    assert np.array_equal(got[layer - 1, r, p, ..., 0], np.broadcast_to(lo, (kv, dim)))
                    assert np.array_equal(got[layer - 1, r, p, ..., 1], np.broadcast_to(hi, (kv, dim)))

    for layer in range(1, layers + 1):
        write(layer, sum((rows(r, 0, n) for r, n in enumerate(lens)), []))
    rpi = torch.arange(len(lens))
    quest.update_prefill_representations_blocks(rpi, i64(lens, cuda), pool, table)
    expect([n // 64 for n in lens])
    # the same chunk by chunk
    quest._reset(0, len(lens))
    mid = [n // 2 for n in lens]
    quest.update_prefill_representations_blocks(rpi, i64(mid, cuda), pool, table)
    quest.update_prefill_representations_blocks(rpi, i64(lens, cuda), pool, table, prefix_lens=i64(mid, cuda), max_new=250)
    expect([n // 64 for n in lens])
    now = list(lens)
    for step in range(66):
        now = [n + 1 for n in now]
        step_layout = quest.decode_step_blocks(rpi, i64(now, cuda), pool, table)
        expect([(n - 1) // 64 for n in now]) if step in (0, 1, 2, 63, 64, 65) else None
        assert step_layout.actual_lens.tolist() == [min(n, 128) for n in now]
        for layer in range(1, layers + 1):
            write(layer, [blocks[r][(n - 1) // 64] * 64 + (n - 1) % 64 for r, n in enumerate(now)])


def test_bounds_of_spoilt_and_missing_blocks(cuda):
    kv, dim = 2, 128
    pool = Fp8TokenToKVPool(6, 1, kv, dim, cuda)
    k = torch.randn(256, kv, dim, device=cuda)
    k[70, 1, 3] = float("nan")
    pool.set_kv_buffer(0, torch.arange(64, 320), k, k)
    quest = QuestAlgorithm(128, 64, cuda)
    quest.init_storage(0, 1, 3, 300, kv, dim)
    table = table_of([[1, 2, 3, 4], [1, 99, -5, 4], [1, 2, 3, 4]], cuda, 9)[:, :4]  # a slice of a wider table
    quest.update_prefill_representations_blocks(i64([0, 1, 7, -1], cuda), i64([256, 9999, 256, 256], cuda), pool, table)
    b = quest.page_k_bounds[0].float()
    assert b[0, 1, 1].isnan().all() and not b[0, 1, 0].isnan().any() and not b[0, [0, 2, 3]].isnan().any()
    assert b[1, [1, 2]].isnan().all() and torch.equal(b[1, [0, 3]], b[0, [0, 3]])
    assert (b[2].abs() == FAR).all() and (b[:2, 4:].abs() == FAR).all()
    with pytest.raises(ValueError, match="length"):
        quest.update_prefill_representations_blocks(i64([0], cuda), i64([1, 2], cuda), pool, table)
    with pytest.raises(ValueError, match="int32"):
        quest.update_prefill_representations_blocks(i64([0], cuda), i64([1], cuda), pool, table.long())
    small = QuestAlgorithm(128, 32, cuda)
    small.init_storage(0, 1, 3, 300, kv, dim)
    with pytest.raises(ValueError, match="64"):
        small.decode_step_blocks(i64([0], cuda), i64([1], cuda), pool, table)
    other = QuestAlgorithm(128, 64, cuda)
    other.init_storage(0, 2, 3, 300, kv, dim)
    with pytest.raises(ValueError, match="layers"):
        other.decode_step_blocks(i64([0], cuda), i64([1], cuda), pool, table)


def test_bounds_refuse_tables_that_are_no_rows(cuda):
    """One row shown as several, whose stride is not the table's width: the kernel would read past it."""
    pool = Fp8TokenToKVPool(6, 1, 2, 128, cuda)
    quest = QuestAlgorithm(128, 64, cuda)
    quest.init_storage(0, 1, 3, 300, 2, 128)
    row = table_of([[1, 2, 3, 4]], cuda, 5)
    lens = i64([0, 1], cuda), i64([65, 65], cuda)
    for bad, said in ((row.expand(3, -1), "overlap"), (row.cpu(), "lies on"), (row[0], "2-D"), (row.t(), "stride")):
        for call in (quest.decode_step_blocks, quest.update_prefill_representations_blocks):
            with pytest.raises(ValueError, match=said):
                call(*lens, pool, bad)
    step = quest.decode_step_blocks(i64([0], cuda), i64([65], cuda), pool, row.expand(1, -1))
    assert step.actual_lens.tolist() == [65] and (quest.page_k_bounds[0, 0, 0] == 0).all()


def test_rescaling_is_exact_down_to_subnormals(cuda):
    """A power of two: growing the scale by 2^m keeps every code whose value stays a multiple of the
    least step."""
    rng = random.Random(2)
    kv, dim = 1, 64
    pool, want = Fp8TokenToKVPool(3, 1, kv, dim, cuda), of.Cache(3, kv, dim)
    x = np.array([[[rng.choice([-1, 1]) * (8 + rng.randint(0, 7)) * 2.0 ** rng.randint(-3, 4) for _ in range(dim)]]], dtype=np.float32)
    for loc, y in ((64, x), (65, x * 0 + 448.0 * 4), (66, x * 0 + 448.0 * 64), (67, x * 0 + 448.0 * 2**20)):
        pool.set_kv_buffer(0, i64([loc], cuda), *(torch.from_numpy(y).to(cuda),) * 2)
        want.write([loc], y, y)
        check(pool, want)
        if loc < 67:
            assert same(pool.get_rows(0, i64([64], cuda))[0].float().cpu().numpy(), x)
