"""Decode attention over the 8-bit block cache, dense and over selected pages, against float64 over
the cache's exact values; the tolerance is oracle.fp8_cache.attend_tolerance's arithmetic."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8_cache as of
from qwenquest_amd.attention.ops import fp8_decode_attention, fp8_decode_plan
from qwenquest_amd.paged import Fp8TokenToKVPool
from qwenquest_amd.quest import QuestAlgorithm

pytestmark = pytest.mark.gpu


def i64(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int64).to(dev)


class Setup:
    """A pool with scattered blocks of random values for every request, and their table."""

    def __init__(self, dev, lens, kv, dim, seed=0, layers=2, layer=1, spare=1, wide=3):
        rng = np.random.default_rng(seed)
        counts = [max(-(-n // 64), 0) + spare for n in lens]
        total = sum(counts) + 1
        ids = (1 + rng.permutation(total - 1)).tolist()
        self.blocks = [[ids.pop() for _ in range(c)] for c in counts]
        self.pool = Fp8TokenToKVPool(total, layers, kv, dim, dev)
        self.layer, self.lens, self.kv, self.dim, self.dev = layer, list(lens), kv, dim, dev
        cols = max(counts) + wide
        wider = torch.zeros((len(lens), cols + 5), dtype=torch.int32)
        for r, b in enumerate(self.blocks):
            wider[r, : len(b)] = torch.tensor(b, dtype=torch.int32)
        self.table = wider.to(dev)[:, :cols]  # columns of a wider table
        gen = torch.Generator(device=dev).manual_seed(seed)
        # every token of every block, those past a context too
        loc = torch.arange(64, total * 64, device=dev)
        shape = (loc.numel(), kv, dim)
        k = torch.empty(shape, device=dev).normal_(generator=gen) + torch.empty((1, kv, dim), device=dev).normal_(generator=gen)
        v = torch.empty(shape, device=dev).normal_(generator=gen)
        size = torch.exp2(torch.randint(-3, 4, (total - 1, kv, 1), device=dev, generator=gen).float()).repeat_interleave(64, 0)
        self.pool.set_kv_buffer(layer, loc, (k * size).to(torch.bfloat16), (v * size.flip(0)).to(torch.bfloat16))

    def rows(self, r, pos):
        b = torch.tensor(self.blocks[r] or [0])
        pos = torch.as_tensor(pos, dtype=torch.int64)
        return b[pos // 64] * 64 + pos % 64

    def values(self, r, pos):
        k, v = self.pool.get_rows(self.layer, self.rows(r, pos), torch.float32)
        return k.double().cpu().numpy(), v.double().cpu().numpy()

    def queries(self, heads, dtype, seed=0, n=None):
        gen = torch.Generator(device=self.dev).manual_seed(100 + seed)
        return torch.empty((n or len(self.lens), heads, self.dim), device=self.dev).normal_(generator=gen).to(dtype)

    def check(self, out, q, scale, positions=None, reqs=None, lens=None):
        bf16 = q.dtype == torch.bfloat16
        assert out.dtype == q.dtype and out.shape == (q.shape[0], q.shape[1] * self.dim)
        got = out.double().cpu().numpy().reshape(q.shape)
        qn = q.double().cpu().numpy()
        for i in range(q.shape[0]):
            r = i if reqs is None else reqs[i]
            n = self.lens[r] if lens is None else lens[i]
            pos = np.arange(n) if positions is None or positions[i] is None else positions[i]
            k, v = self.values(r, pos)
            want, spread, size = of.attend(qn[i], k, v, scale)
            tol = of.attend_tolerance(want, spread, size, len(pos), self.dim, bf16, 16 if bf16 else 24)
            err = np.abs(got[i] - want)
            assert (err <= tol).all(), f"request {i} ({len(pos)} tokens): off by {(err / tol).max():.2f} tolerances"


RAGGED = [1, 0, 63, 64, 65, 128, 700, 5, 129, 2000]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv, dim", [(32, 4, 128), (1, 1, 128), (5, 1, 64), (16, 8, 128), (48, 3, 64), (17, 1, 128),
                                            (80, 2, 64), (7, 7, 128), (66, 2, 128)])
def test_ragged_batches(cuda, heads, kv, dim, dtype):
    s = Setup(cuda, RAGGED, kv, dim, seed=heads)
    q = s.queries(heads, dtype)
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, torch.arange(len(RAGGED)), i64(RAGGED, cuda), dim**-0.5)
    s.check(out, q, dim**-0.5)
    assert not out[1].any()  # an empty context


@pytest.mark.parametrize("lens", [[70000], [1], [20000, 1, 1, 19999], [64] * 300, [1 + i % 130 for i in range(1500)],
                                  [3000] * 40])
def test_divisions_of_the_work(cuda, lens):
    """One request in many slices, many in one, more than the plan's threads."""
    s = Setup(cuda, lens, 2, 64, seed=len(lens))
    q = s.queries(6, torch.bfloat16)
    args = (s.pool, s.layer, s.table, torch.arange(len(lens)), i64(lens, cuda), 0.125)
    out = fp8_decode_attention(q, *args)
    s.check(out, q, 0.125)
    assert torch.equal(out, fp8_decode_attention(q, *args))  # no order of arrival in the sums


@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0, 1e-30])
def test_any_scale(cuda, scale):
    s = Setup(cuda, [300, 1, 64], 2, 128, seed=3)
    q = s.queries(8, torch.float32)
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, torch.arange(3), i64([300, 1, 64], cuda), scale)
    s.check(out, q, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
def test_weights_keep_their_bits(cuda, dim, dtype):
    """A sum in which values cancel, so that a weight's lower bits decide: head h's token 0 weighs
    exp(-a) against 1 of tokens 1 and 2, which hold -exp(-a) to 8 bits in channel h.

    Roundings: the score's one product is exact, its scaling to a power of two and back a few times 2^-24
    of |t| <= 2, so that a weight is off by under 2^-21 of itself, the exponential's last place included;
    pieces of 24 bits add 2^-24, sums of three terms as much each.  All of it under 2^-20 of
    sum p |v|; a weight of 16 bits alone is off by up to 2^-15."""
    heads = 16
    a = (0.3 + torch.arange(heads) / 12.0).to(torch.bfloat16).double()
    pool = Fp8TokenToKVPool(2, 1, 1, dim, cuda)
    k, v = torch.zeros(3, 1, dim, dtype=torch.float64), torch.zeros(3, 1, dim, dtype=torch.float64)
    k[0, 0, 0] = -1.0
    v[0, 0, :heads] = 1.0
    p = torch.exp(-a)
    first = torch.from_numpy(of.round_e4m3(p.numpy()))
    v[1, 0, :heads] = -first
    v[2, 0, :heads] = -torch.from_numpy(of.round_e4m3((p - first).numpy() * 64) / 64)
    pool.set_kv_buffer(0, torch.arange(64, 67), k.float().to(cuda), v.float().to(cuda))
    got = pool.get_rows(0, torch.arange(64, 67), torch.float32)
    assert torch.equal(got[0].cpu().double(), k) and torch.equal(got[1].cpu().double(), v)  # exact in 8 bits
    q = torch.zeros(1, heads, dim, dtype=torch.float64)
    q[0, :, 0] = a
    table = torch.tensor([[1]], dtype=torch.int32, device=cuda)
    out = fp8_decode_attention(q.to(cuda, dtype), pool, 0, table, i64([0], cuda), i64([3], cuda), 1.0)
    got = out.view(heads, dim).double().cpu().diagonal()
    total = p + 2
    want = (p + v[1, 0, :heads] + v[2, 0, :heads]) / total
    spread = (p + v[1:, 0, :heads].abs().sum(0)) / total
    assert (want.abs() < spread * 2.0**-8).all() and (want.abs() > spread * 2.0**-20).sum() > heads // 2
    half = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-24
    err = (got - want).abs()
    assert (err <= half * want.abs() + 2.0**-20 * spread).all(), (err / (half * want.abs() + 2.0**-20 * spread)).max()


def picked(rng, n, top_k, pages=None):
    """A selection as retrieve_topk lays it out: pages in any order, expanded, then the recent window."""
    k = top_k // 64 - 1
    pages = rng.permutation(n // 64)[:k] if pages is None else np.asarray(pages)
    return np.concatenate([(pages[:, None] * 64 + np.arange(64)).reshape(-1), np.arange(n - 64, n)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top_k", [64, 128, 512, 2048])
def test_selected_pages(cuda, top_k, dtype):
    """Long requests by their pages and window (overlapping or not), short ones densely."""
    rng = np.random.default_rng(top_k)
    lens = [top_k + 1, top_k, top_k + 64, top_k + 63, 5000, 0, 1, 5056, top_k - 1, 5121]
    s = Setup(cuda, lens, 2, 128, seed=top_k)
    q = s.queries(10, dtype)
    positions = np.zeros((len(lens) + 1, top_k), dtype=np.int32)
    want = []
    for i, n in enumerate(lens):
        want.append(picked(rng, n, top_k) if n > top_k else None)
        if n > top_k:
            positions[i] = want[-1]
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, torch.arange(len(lens)), i64(lens, cuda), 0.08,
                               positions=torch.from_numpy(positions).to(cuda), top_k=top_k)
    s.check(out, q, 0.08, positions=want)


def test_a_page_selected_twice_counts_twice(cuda):
    s = Setup(cuda, [1000], 1, 64)
    q = s.queries(3, torch.float32)
    pos = picked(None, 1000, 256, pages=[4, 4, 0])
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, i64([0], cuda), i64([1000], cuda), 0.2,
                               positions=torch.from_numpy(pos[None].astype(np.int32)).to(cuda), top_k=256)
    s.check(out, q, 0.2, positions=[pos])


def test_requests_and_blocks_that_are_not_there(cuda):
    """NaN for them alone; a request listed twice is attended twice."""
    lens = [200, 300, 64]
    s = Setup(cuda, lens, 2, 128)
    reqs = [0, 3, 1, -1, 2, 0, 1 << 40]
    q = s.queries(4, torch.bfloat16, n=len(reqs))
    n = [200, 10, 300, 10, 0, 130, 5]
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, i64(reqs, cuda), i64(n, cuda), 0.1)
    assert out[[1, 3, 6]].isnan().all()
    ok = [0, 2, 4, 5]
    s.check(out[ok], q[ok], 0.1, reqs=[reqs[i] for i in ok], lens=[n[i] for i in ok])
    # a context past its blocks, a block outside the pool, a page outside the table
    out = fp8_decode_attention(q[:3], s.pool, s.layer, s.table, torch.arange(3), i64([200, 300 + 128, 64], cuda), 0.1)
    assert out[1].isnan().all() and not out[[0, 2]].isnan().any()
    table = s.table.clone()
    table[0, 1], table[2, 0] = s.pool.num_blocks, -7
    out = fp8_decode_attention(q[:3], s.pool, s.layer, table, torch.arange(3), i64(lens, cuda), 0.1)
    assert out[[0, 2]].isnan().all() and not out[1].isnan().any()
    positions = torch.zeros((3, 128), dtype=torch.int32, device=cuda)
    positions[1] = 64 * 100000
    positions[0] = -64
    out = fp8_decode_attention(q[:3], s.pool, s.layer, s.table, torch.arange(3), i64(lens, cuda), 0.1, positions=positions,
                               top_k=128)
    assert out[:2].isnan().all() and not out[2].isnan().any()
    # lengths past the table's width are cut to it, negative ones are empty
    full = s.table.shape[1] * 64
    s.table[0] = s.table[0, 0]
    out = fp8_decode_attention(q[:2], s.pool, s.layer, s.table, i64([0, 1], cuda), i64([1 << 50, -3], cuda), 0.1)
    assert not out[0].isnan().any() and not out[1].any()
    again = fp8_decode_attention(q[:1], s.pool, s.layer, s.table, i64([0], cuda), i64([full], cuda), 0.1)
    assert torch.allclose(out[:1].float(), again.float(), rtol=2.0**-7, atol=1e-5)


def test_spoilt_values_reach_those_who_attend_them(cuda):
    """A block with a value that is not finite: NaN for the requests and heads that attend it, nothing
    for the others, nor for a selection without it; nothing of what lies behind a context."""
    lens = [200, 200, 500]
    s = Setup(cuda, lens, 2, 64)
    for which, (r, p, h) in enumerate(((0, 100, 0), (1, 130, 1), (2, 490, 0))):
        x = [torch.zeros(1, 2, 64, device=cuda) for _ in range(2)]
        x[which % 2][0, h, 3] = float("inf")
        s.pool.set_kv_buffer(s.layer, s.rows(r, [p]), *x)
    q = s.queries(4, torch.bfloat16)
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, torch.arange(3), i64(lens, cuda), 0.1).view(3, 4, 64)
    assert out[0, :2].isnan().all() and not out[0, 2:].isnan().any()
    assert out[1, 2:].isnan().all() and not out[1, :2].isnan().any()
    assert out[2, :2].isnan().all() and not out[2, 2:].isnan().any()
    short = [60, 128, 448]  # before the spoilt blocks
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, torch.arange(3), i64(short, cuda), 0.1)
    s.check(out, q, 0.1, lens=short)
    pos = [picked(None, n, 128, pages=[0]) for n in (200, 200, 447)]
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, torch.arange(3), i64([200, 200, 447], cuda), 0.1,
                               positions=torch.from_numpy(np.stack(pos).astype(np.int32)).to(cuda), top_k=128)
    assert not out[[0, 2]].isnan().any()  # block 1 of request 0 is not among them, block 7 of request 2 not begun on
    # tokens behind the context, in its last block: larger than anything, and without weight
    x = torch.full((1, 2, 64), 1e30, device=cuda)
    clean = Setup(cuda, [100], 2, 64, seed=9)
    clean.pool.set_kv_buffer(1, clean.rows(0, [100]), x, x)
    q1 = q[:1]
    out = fp8_decode_attention(q1, clean.pool, 1, clean.table, i64([0], cuda), i64([100], cuda), 0.1)
    clean.check(out, q1, 0.1)


def test_queries_that_are_not_finite(cuda):
    s = Setup(cuda, [200, 200], 2, 128)
    for dtype in (torch.bfloat16, torch.float32):
        q = s.queries(4, dtype)
        q[0, 1, 5] = float("nan")
        q[0, 2, 7] = float("inf")
        out = fp8_decode_attention(q, s.pool, s.layer, s.table, torch.arange(2), i64([200, 200], cuda), 0.1).view(2, 4, 128)
        assert out[0, 1:3].isnan().all() and not out[0, [0, 3]].isnan().any() and not out[1].isnan().any()


def test_new_tokens_are_stored_and_attended(cuda):
    lens = [65, 1, 300, 128]
    s = Setup(cuda, lens, 2, 128, seed=5)
    want = Setup(cuda, lens, 2, 128, seed=5)
    q = s.queries(8, torch.bfloat16)
    k, v = (torch.randn(4, 2, 128, device=cuda, dtype=torch.bfloat16) * 9 for _ in range(2))
    loc = torch.cat([s.rows(r, [n - 1]) for r, n in enumerate(lens)])
    loc[3] = 0  # a padded entry stores nothing
    out = fp8_decode_attention(q, s.pool, s.layer, s.table, torch.arange(4), i64(lens, cuda), 0.1, new=(loc, k, v))
    want.pool.set_kv_buffer(want.layer, loc, k, v)
    assert torch.equal(s.pool.k_codes, want.pool.k_codes) and torch.equal(s.pool.v_scale, want.pool.v_scale)
    s.check(out, q, 0.1)


@pytest.mark.parametrize("heads, kv, dim, dtype, lens", [
    (32, 4, 128, torch.bfloat16, [1, 64, 65, 128, 0, 700, 4097, 5000, 2]), (3, 3, 64, torch.float32, [129, 192, 1, 1000]),
    (16, 1, 128, torch.float32, [1 + i % 70 for i in range(600)]), (34, 2, 64, torch.bfloat16, [100, 64, 1]),
    (4, 1, 64, torch.bfloat16, [1 + i * 37 % 65 for i in range(2500)]), (8, 4, 128, torch.bfloat16, [20000]),
    (8, 4, 128, torch.bfloat16, [64 * 40] * 48)])
def test_a_step_divided_once_for_its_layers(cuda, heads, kv, dim, dtype, lens):
    """Layers of one plan leave the cache and the answers, to the bit, that calls without one do: new
    tokens that begin a block, make its scale grow, are not finite or are nobody's (block 0)."""
    ours, want = (Setup(cuda, lens, kv, dim, seed=7, layer=1) for _ in range(2))
    n, reqs = i64(lens, cuda), torch.arange(len(lens), device=cuda)
    loc = torch.cat([s_rows for s_rows in (ours.rows(r, [max(m, 1) - 1]) for r, m in enumerate(lens))])
    loc[2::11] = 0
    gen = torch.Generator(device=cuda).manual_seed(3)
    for step in range(3):  # the same division three times over
        plan = fp8_decode_plan(ours.pool, ours.table, reqs, n) if step != 1 else plan
        for layer in (0, 1):  # layer 0: nothing there yet
            q = ours.queries(heads, dtype, 10 * step + layer)
            k, v = (torch.randn(len(lens), kv, dim, device=cuda, generator=gen) for _ in range(2))
            k[::3] *= 2.0 ** (3 * step)
            v[1::4] *= 2.0 ** (3 * step)
            k[5::13, 0, 3], v[7::17, kv - 1, 60] = float("nan"), float("inf")
            k, v = k.to(dtype), v.to(dtype)
            a = fp8_decode_attention(q, ours.pool, layer, ours.table, reqs, n, 0.1, new=(loc, k, v), plan=plan)
            b = fp8_decode_attention(q, want.pool, layer, want.table, reqs, n, 0.1, new=(loc, k, v))
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) or torch.equal(a.isnan(), b.isnan())
            assert torch.equal(a.nan_to_num(), b.nan_to_num())
            for x in ("k_codes", "v_codes", "k_scale", "v_scale"):
                assert torch.equal(getattr(ours.pool, x)[layer].view(torch.uint8)[1:], getattr(want.pool, x)[layer].view(torch.uint8)[1:]), x
    a = fp8_decode_attention(q, ours.pool, 1, ours.table, reqs, n, 0.1, plan=plan)  # nothing to store
    assert torch.equal(a.nan_to_num(), b.nan_to_num())


def test_a_plan_of_other_lengths_answers_nothing_wrong(cuda):
    """Lengths and requests that change behind the plan: the right answer or NaN."""
    lens = [500, 64, 3000, 1, 200, 700]
    s = Setup(cuda, lens, 2, 128, spare=4)
    q, n, reqs = s.queries(8, torch.bfloat16), i64(lens, cuda), torch.arange(6, device=cuda)
    plan = fp8_decode_plan(s.pool, s.table, reqs, n)
    lone = [fp8_decode_plan(s.pool, s.table, reqs[i : i + 1], n[i : i + 1]) for i in range(6)]
    changes = [(n + 1, reqs), (n + 64, reqs), (n - 1, reqs), (n // 2, reqs), (n.flip(0), reqs), (n * 0, reqs), (n, reqs.flip(0))]
    for m, r in changes:
        want = fp8_decode_attention(q, s.pool, s.layer, s.table, r, m, 0.1)
        got = fp8_decode_attention(q, s.pool, s.layer, s.table, r, m, 0.1, plan=plan)
        ok = got.isnan().all(1) | ((got.float() - want.float()).abs() <= 2**-7 * want.float().abs().amax(1, keepdim=True)).all(1)
        assert ok.all(), (m, r, ok)
        for i in range(6):
            one = fp8_decode_attention(q[i : i + 1], s.pool, s.layer, s.table, r[i : i + 1], m[i : i + 1], 0.1, plan=lone[i])
            assert one.isnan().all() or ((m[i] == n[i]) & (r[i] == reqs[i]))
    again = fp8_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1, plan=plan)
    s.check(again, q, 0.1)


def test_a_plan_is_checked(cuda):
    s = Setup(cuda, [100, 100], 2, 64)
    q, r, n = s.queries(4, torch.bfloat16), torch.arange(2), i64([100, 100], cuda)
    plan = fp8_decode_plan(s.pool, s.table, r, n)
    others = i64(range(3), cuda) % 2
    more = fp8_decode_plan(s.pool, s.table, others, n[:1].repeat(3))
    wider = fp8_decode_plan(Setup(cuda, [100, 100], 4, 64).pool, s.table, r, n)
    for bad in (more, wider, plan._replace(workspace=plan.workspace.cpu())):
        with pytest.raises(ValueError, match="plan"):
            fp8_decode_attention(q, s.pool, s.layer, s.table, r, n, 0.1, plan=bad)
    with pytest.raises(ValueError, match="selected pages"):
        fp8_decode_attention(q, s.pool, s.layer, s.table, r, n, 0.1, plan=plan, top_k=64,
                             positions=torch.zeros(2, 64, dtype=torch.int32, device=cuda))
    s.check(fp8_decode_attention(q, s.pool, s.layer, s.table, r, n, 0.1, plan=plan), q, 0.1)
    assert fp8_decode_plan(s.pool, s.table, r[:0], n[:0]).bs == 0


@pytest.mark.parametrize("heads, kv, dim, dtype", [(32, 4, 128, torch.bfloat16), (3, 3, 64, torch.float32), (10, 1, 128, torch.bfloat16)])
def test_a_plan_of_another_batch_answers_nan(cuda, heads, kv, dim, dtype):
    """Plans of other requests, or of selections, that do not show it: every output written, and NaN; the
    cache as it was.  Those that show it are refused."""
    lens = [500, 64, 0, 1300]
    s = Setup(cuda, lens, kv, dim)
    q, reqs, n = s.queries(heads, dtype), torch.arange(4, device=cuda), i64(lens, cuda)
    rows = torch.cat([s.rows(r, [max(m, 1) - 1]) for r, m in enumerate(lens)])
    new = (rows, *(torch.randn(4, kv, dim, device=cuda, dtype=dtype) for _ in range(2)))
    few = fp8_decode_plan(s.pool, s.table, reqs[:3], n[:3])
    quest = QuestAlgorithm(128, 64, cuda)
    quest.init_storage(0, 2, 4, s.table.shape[1] * 64, kv, dim)
    sparse = quest.decode_step_blocks(reqs, n, s.pool, s.table).plan
    before = s.pool.k_codes.clone(), s.pool.v_scale.clone()
    for plan in (few._replace(bs=4), sparse._replace(top_k=0)):
        junk = torch.full((4, heads * dim), 7.0, device=cuda, dtype=dtype)  # what the allocator may hand out again
        del junk
        out = fp8_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1, new=new, plan=plan)
        assert out.isnan().all()
        assert torch.equal(before[0], s.pool.k_codes) and torch.equal(before[1], s.pool.v_scale)
    for plan in (few, sparse):
        with pytest.raises(ValueError, match="plan"):
            fp8_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1, plan=plan)
    s.check(fp8_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1, plan=fp8_decode_plan(s.pool, s.table, reqs, n)), q, 0.1)


def test_arguments_are_checked(cuda):
    s = Setup(cuda, [100, 100], 2, 64)
    q, r, n = s.queries(4, torch.bfloat16), torch.arange(2), i64([100, 100], cuda)

    def call(q=q, table=s.table, r=r, n=n, **kw):
        return fp8_decode_attention(q, s.pool, s.layer, table, r, n, 0.1, **kw)

    for bad, said in ((dict(q=q[:, :3]), "divisible"), (dict(q=q.half()), "dtype"), (dict(q=q[..., :32]), "heads, 64"),
                      (dict(q=q.cpu()), "lies on"), (dict(table=s.table.long()), "int32"), (dict(table=s.table[0]), "2-D"),
                      (dict(table=s.table.cpu()), "lies on"), (dict(r=r[:1]), "entries"), (dict(n=i64([1, 2, 3], cuda)), "entries"),
                      (dict(positions=torch.zeros(2, 128, device=cuda), top_k=128), "positions"),
                      (dict(positions=torch.zeros(2, 64, dtype=torch.int32, device=cuda), top_k=128), "positions"),
                      (dict(positions=torch.zeros(2, 100, dtype=torch.int32, device=cuda), top_k=100), "multiple"),
                      (dict(new=(r, torch.zeros(1, 2, 64), torch.zeros(1, 2, 64))), "rows")):
        with pytest.raises(ValueError, match=said):
            call(**bad)
    flat = call(q=q.view(2, -1))
    strided = torch.zeros(2, 8, 64, device=cuda, dtype=torch.bfloat16)
    strided[:, ::2] = q
    assert torch.equal(flat, call(q=strided[:, ::2])) and torch.equal(flat, call(r=r.int(), n=n.int().cpu()))
    assert call(q=q[:0], r=r[:0], n=n[:0]).shape == (0, 256)


def test_replayed_graphs_with_growing_lengths(cuda):
    """Two captured calls of different shapes, replayed in turn while lengths change in place and other
    batches run eagerly between them."""
    lens = [500, 2000, 64]
    s = Setup(cuda, lens, 2, 128)
    qa, qb = s.queries(8, torch.bfloat16, 1), s.queries(2, torch.float32, 2)
    na, nb = i64([100, 1, 30], cuda), i64([64, 1000, 2], cuda)
    reqs = torch.arange(3, device=cuda)

    def a():
        return fp8_decode_attention(qa, s.pool, s.layer, s.table, reqs, na, 0.1)

    def b():
        return fp8_decode_attention(qb, s.pool, s.layer, s.table, reqs, nb, 0.1)

    a(), b()
    torch.cuda.synchronize()
    graphs = []
    for f in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, out))
    for step in range(4):
        na += i64([90, 450, 8], cuda)
        nb -= i64([9, 200, 0], cuda)
        for g, _ in graphs:
            g.replay()
        fp8_decode_attention(s.queries(8, torch.bfloat16, 7), s.pool, s.layer, s.table, reqs, i64(lens, cuda), 0.1)
        assert torch.equal(graphs[0][1], a()) and torch.equal(graphs[1][1], b())
        s.check(graphs[0][1], qa, 0.1, lens=na.tolist())
        s.check(graphs[1][1], qb, 0.1, lens=nb.tolist())


def test_two_streams_at_once(cuda):
    lens = [6000, 40, 900]
    s = Setup(cuda, lens, 2, 128)
    qs = [s.queries(8, torch.bfloat16, i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    n, reqs = i64(lens, cuda), torch.arange(3, device=cuda)
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for st, q in zip(streams, qs):
            with torch.cuda.stream(st):
                outs.append(fp8_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, outs[i % 2])
    for i in range(2):
        s.check(outs[i], qs[i], 0.1)
