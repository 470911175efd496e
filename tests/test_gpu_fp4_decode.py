"""Decode attention over the 4-bit block cache, dense and over selected pages, against float64 over
the cache's exact values; the tolerance is oracle.fp8_cache.attend_tolerance's arithmetic, which
counts the same roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp4_cache as o4
from oracle import fp8_cache as of
from qwenquest_amd.attention.ops import fp4_decode_attention, fp4_decode_plan, fp8_decode_attention
from qwenquest_amd.paged import Fp4TokenToKVPool
from qwenquest_amd.quest import QuestAlgorithm
from tests.test_gpu_fp8_decode import RAGGED, i64, picked
from tests.test_gpu_fp8_decode import Setup as Setup8

pytestmark = pytest.mark.gpu


class Setup(Setup8):
    """A 4-bit pool with scattered blocks of random values for every request, and their table."""

    def __init__(self, dev, lens, kv, dim, seed=0, layers=2, layer=1, spare=1, wide=3):
        rng = np.random.default_rng(seed)
        counts = [-(-n // 64) + spare for n in lens]
        total = sum(counts) + 1
        ids = (1 + rng.permutation(total - 1)).tolist()
        self.blocks = [[ids.pop() for _ in range(c)] for c in counts]
        self.pool = Fp4TokenToKVPool(total, layers, kv, dim, dev)
        self.layer, self.lens, self.kv, self.dim, self.dev = layer, list(lens), kv, dim, dev
        cols = max(counts) + wide
        wider = torch.zeros((len(lens), cols + 5), dtype=torch.int32)
        for r, b in enumerate(self.blocks):
            wider[r, : len(b)] = torch.tensor(b, dtype=torch.int32)
        self.table = wider.to(dev)[:, :cols]  # columns of a wider table
        gen = torch.Generator(device=dev).manual_seed(seed)
        # every token of every block, those past a context too; sizes differ by token and by channel
        loc = torch.arange(64, total * 64, device=dev)
        shape = (loc.numel(), kv, dim)
        k = torch.empty(shape, device=dev).normal_(generator=gen) + torch.empty((1, kv, dim), device=dev).normal_(generator=gen) * 2
        v = torch.empty(shape, device=dev).normal_(generator=gen)
        size = torch.exp2(torch.randint(-3, 4, (loc.numel(), kv, 1), device=dev, generator=gen).float())
        self.pool.set_kv_buffer(layer, loc, k.to(torch.bfloat16), (v * size).to(torch.bfloat16))


    def check(self, out, q, scale, positions=None, reqs=None, lens=None):
        """The 8-bit cache's tolerance and what underflows: 4-bit codes are often exactly 0, so that a channel may hold
        nothing of the tokens that weigh most, and its output be of the size of float32's least numbers.  A weight
        under 2^-126 is 0 (off by that times its value, at most |v|), as is each of its three pieces (times a code of 6
        at most), and a sum of 32 products (of n / 32), where the weights' sum is 1 at least: in all
        n 2^-126 (max |v| + 3 * 6 + 1)."""
        bf16 = q.dtype == torch.bfloat16
        assert out.dtype == q.dtype and out.shape == (q.shape[0], q.shape[1] * self.dim)
        got, qn = out.double().cpu().numpy().reshape(q.shape), q.double().cpu().numpy()
        for i in range(q.shape[0]):
            r = i if reqs is None else reqs[i]
            n = self.lens[r] if lens is None else lens[i]
            pos = np.arange(n) if positions is None or positions[i] is None else positions[i]
            k, v = self.values(r, pos)
            want, spread, size = of.attend(qn[i], k, v, scale)
            tol = of.attend_tolerance(want, spread, size, len(pos), self.dim, bf16, 16 if bf16 else 24)
            tol += len(pos) * 2.0**-126 * (np.abs(v).max(initial=0.0) + 19)
            err = np.abs(got[i] - want)
            assert (err <= tol).all(), f"request {i} ({len(pos)} tokens): off by {(err / tol).max():.2f} tolerances"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv, dim", [(32, 4, 128), (1, 1, 128), (5, 1, 64), (16, 8, 128), (48, 3, 64), (17, 1, 128),
                                            (80, 2, 64), (7, 7, 128), (66, 2, 128)])
def test_ragged_batches(cuda, heads, kv, dim, dtype):
    s = Setup(cuda, RAGGED, kv, dim, seed=heads)
    q = s.queries(heads, dtype)
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(len(RAGGED)), i64(RAGGED, cuda), dim**-0.5)
    s.check(out, q, dim**-0.5)
    assert not out[1].any()  # an empty context


@pytest.mark.parametrize("lens", [[70000], [1], [20000, 1, 1, 19999], [64] * 300, [1 + i % 130 for i in range(1500)],
                                  [3000] * 40])
def test_divisions_of_the_work(cuda, lens):
    """One request in many slices, many in one, more than the plan's threads."""
    s = Setup(cuda, lens, 2, 64, seed=len(lens))
    q = s.queries(6, torch.bfloat16)
    args = (s.pool, s.layer, s.table, torch.arange(len(lens)), i64(lens, cuda), 0.125)
    out = fp4_decode_attention(q, *args)
    s.check(out, q, 0.125)
    assert torch.equal(out, fp4_decode_attention(q, *args))  # no order of arrival in the sums


@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0, 1e-30])
def test_any_scale(cuda, scale):
    s = Setup(cuda, [300, 1, 64], 2, 128, seed=3)
    q = s.queries(8, torch.float32)
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(3), i64([300, 1, 64], cuda), scale)
    s.check(out, q, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
def test_weights_keep_their_bits(cuda, dim, dtype):
    """A sum in which values cancel, so that a weight's lower bits decide: head h's token 0 weighs
    exp(-a) against 1 of the others, which hold -exp(-a) in channel h, 2 bits at a time.

    Roundings: the score's one product is exact, its scaling to a power of two and back a few times 2^-24
    of |t| <= 2, so that a weight is off by under 2^-21 of itself, the exponential's last place included;
    pieces of 24 bits add 2^-24, sums of up to nine terms eight times half a step of the largest, 2^-21.  All of it
    under 2^-19 of sum p |v|; a weight of 11 bits alone is off by up to 2^-10."""
    heads, n = 16, 9
    a = (0.3 + torch.arange(heads) / 12.0).to(torch.bfloat16).double()
    pool = Fp4TokenToKVPool(2, 1, 1, dim, cuda)
    k, v = torch.zeros(n, 1, dim, dtype=torch.float64), torch.zeros(n, 1, dim, dtype=torch.float64)
    k[0, 0, 0] = -1.0
    v[0, 0, :heads] = 1.0
    p = torch.exp(-a)
    left = p.clone()
    for i in range(1, n):  # token i holds what its scale of 2^(-2 i) can say of what is left
        e = 2.0 ** (-2 * i)
        part = torch.from_numpy(o4.round_e2m1((left / e).clamp(max=6).numpy())) * e
        v[i, 0, :heads] = -part
        v[i, 0, heads] = 4 * e  # pins the scale
        left = left - part
    pool.set_kv_buffer(0, torch.arange(64, 64 + n), k.float().to(cuda), v.float().to(cuda))
    got = pool.get_rows(0, torch.arange(64, 64 + n), torch.float32)
    assert torch.equal(got[0].cpu().double(), k) and torch.equal(got[1].cpu().double(), v)  # exact in 4 bits
    q = torch.zeros(1, heads, dim, dtype=torch.float64)
    q[0, :, 0] = a
    table = torch.tensor([[1]], dtype=torch.int32, device=cuda)
    out = fp4_decode_attention(q.to(cuda, dtype), pool, 0, table, i64([0], cuda), i64([n], cuda), 1.0)
    got = out.view(heads, dim).double().cpu().diagonal()
    total = p + n - 1
    want, spread = left / total, (p + v[1:, 0, :heads].abs().sum(0)) / total
    assert (want.abs() < spread * 2.0**-9).all()
    half = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-24
    err = (got - want).abs()
    assert (err <= half * want.abs() + 2.0**-19 * spread).all(), (err / (half * want.abs() + 2.0**-19 * spread)).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top_k, kv, dim", [(64, 2, 128), (128, 2, 128), (512, 3, 64), (2048, 2, 128)])
def test_selected_pages(cuda, top_k, kv, dim, dtype):
    """Long requests by their pages and window (overlapping or not), short ones densely."""
    rng = np.random.default_rng(top_k)
    lens = [top_k + 1, top_k, top_k + 64, top_k + 63, 5000, 0, 1, 5056, top_k - 1, 5121]
    s = Setup(cuda, lens, kv, dim, seed=top_k)
    q = s.queries(5 * kv, dtype)
    positions = np.zeros((len(lens) + 1, top_k), dtype=np.int32)
    want = []
    for i, n in enumerate(lens):
        want.append(picked(rng, n, top_k) if n > top_k else None)
        if n > top_k:
            positions[i] = want[-1]
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(len(lens)), i64(lens, cuda), 0.08,
                               positions=torch.from_numpy(positions).to(cuda), top_k=top_k)
    s.check(out, q, 0.08, positions=want)


@pytest.mark.parametrize("dim", [64, 128])
def test_windows_at_every_place(cuda, dim):
    """The last 64 tokens from every place of two blocks."""
    lens = [192 + i for i in range(1, 66)]
    s = Setup(cuda, lens, 1, dim, seed=1)
    q = s.queries(3, torch.float32)
    positions = np.stack([picked(None, n, 128, pages=[0]) for n in lens])
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(len(lens)), i64(lens, cuda), 0.1,
                               positions=torch.from_numpy(positions.astype(np.int32)).to(cuda), top_k=128)
    s.check(out, q, 0.1, positions=list(positions))


def test_a_page_selected_twice_counts_twice(cuda):
    s = Setup(cuda, [1000], 1, 64)
    q = s.queries(3, torch.float32)
    pos = picked(None, 1000, 256, pages=[4, 4, 0])
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, i64([0], cuda), i64([1000], cuda), 0.2,
                               positions=torch.from_numpy(pos[None].astype(np.int32)).to(cuda), top_k=256)
    s.check(out, q, 0.2, positions=[pos])


def test_requests_and_blocks_that_are_not_there(cuda):
    """NaN for them alone; a request listed twice is attended twice."""
    lens = [200, 300, 64]
    s = Setup(cuda, lens, 2, 128)
    reqs = [0, 3, 1, -1, 2, 0, 1 << 40]
    q = s.queries(4, torch.bfloat16, n=len(reqs))
    n = [200, 10, 300, 10, 0, 130, 5]
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, i64(reqs, cuda), i64(n, cuda), 0.1)
    assert out[[1, 3, 6]].isnan().all()
    ok = [0, 2, 4, 5]
    s.check(out[ok], q[ok], 0.1, reqs=[reqs[i] for i in ok], lens=[n[i] for i in ok])
    # a context past its blocks, a block outside the pool, a page outside the table
    out = fp4_decode_attention(q[:3], s.pool, s.layer, s.table, torch.arange(3), i64([200, 300 + 128, 64], cuda), 0.1)
    assert out[1].isnan().all() and not out[[0, 2]].isnan().any()
    table = s.table.clone()
    table[0, 1], table[2, 0] = s.pool.num_blocks, -7
    out = fp4_decode_attention(q[:3], s.pool, s.layer, table, torch.arange(3), i64(lens, cuda), 0.1)
    assert out[[0, 2]].isnan().all() and not out[1].isnan().any()
    positions = torch.zeros((3, 128), dtype=torch.int32, device=cuda)
    positions[1] = 64 * 100000
    positions[0] = -64
    out = fp4_decode_attention(q[:3], s.pool, s.layer, s.table, torch.arange(3), i64(lens, cuda), 0.1, positions=positions,
                               top_k=128)
    assert out[:2].isnan().all() and not out[2].isnan().any()
    # lengths past the table's width are cut to it, negative ones are empty
    full = s.table.shape[1] * 64
    s.table[0] = s.table[0, 0]
    out = fp4_decode_attention(q[:2], s.pool, s.layer, s.table, i64([0, 1], cuda), i64([1 << 50, -3], cuda), 0.1)
    assert not out[0].isnan().any() and not out[1].any()
    again = fp4_decode_attention(q[:1], s.pool, s.layer, s.table, i64([0], cuda), i64([full], cuda), 0.1)
    assert torch.allclose(out[:1].float(), again.float(), rtol=2.0**-7, atol=1e-5)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lost_tokens_reach_those_who_attend_them(cuda, dim, dtype):
    """A token with a value that is not finite: NaN for the requests and heads that attend it, whatever it
    weighs, nothing for the others, nor for a selection without it, nor behind a context."""
    lens = [200, 200, 500]
    s = Setup(cuda, lens, 2, dim)
    for which, (r, p, h) in enumerate(((0, 100, 0), (1, 130, 1), (2, 490, 0))):
        x = [torch.zeros(1, 2, dim, device=cuda) for _ in range(2)]
        x[which % 2][0, h, 3] = float("inf")
        s.pool.set_kv_buffer(s.layer, s.rows(r, [p]), *x)
    q = s.queries(4, dtype)
    for scale in (0.1, 30.0):
        out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(3), i64(lens, cuda), scale).view(3, 4, dim)
        assert out[0, :2].isnan().all() and not out[0, 2:].isnan().any()
        assert out[1, 2:].isnan().all() and not out[1, :2].isnan().any()
        assert out[2, :2].isnan().all() and not out[2, 2:].isnan().any()
    short = [100, 130, 490]  # up to the lost tokens, which lie right behind
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(3), i64(short, cuda), 0.1)
    s.check(out, q, 0.1, lens=short)
    n = [229, 200, 490]
    pos = [picked(None, m, 128, pages=[0]) for m in n]  # windows 165 .., 136 .., 426 ..
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(3), i64(n, cuda), 0.1,
                               positions=torch.from_numpy(np.stack(pos).astype(np.int32)).to(cuda), top_k=128)
    s.check(out, q, 0.1, positions=pos, lens=n)


def test_queries_that_are_not_finite(cuda):
    s = Setup(cuda, [200, 200], 2, 128)
    for dtype in (torch.bfloat16, torch.float32):
        q = s.queries(4, dtype)
        q[0, 1, 5] = float("nan")
        q[0, 2, 7] = float("inf")
        out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(2), i64([200, 200], cuda), 0.1).view(2, 4, 128)
        assert out[0, 1:3].isnan().all() and not out[0, [0, 3]].isnan().any() and not out[1].isnan().any()


@pytest.mark.parametrize("sizes", [(2.0**-40, 2.0**40), (2.0**55, 1.0), (2.0**-46, 2.0**-46)])
def test_values_of_very_different_size(cuda, sizes):
    s = Setup(cuda, [300, 70], 2, 64)
    for r, n in enumerate(s.lens):
        x = torch.randn(n, 2, 64, device=cuda)
        v = torch.randn(n, 2, 64, device=cuda) * torch.tensor(sizes, device=cuda)[torch.arange(n, device=cuda) % 2][:, None, None]
        s.pool.set_kv_buffer(s.layer, s.rows(r, np.arange(n)), x, v)
    for dtype in (torch.bfloat16, torch.float32):
        q = s.queries(4, dtype)
        out = fp4_decode_attention(q, s.pool, s.layer, s.table, torch.arange(2), i64(s.lens, cuda), 0.3)
        s.check(out, q, 0.3)


@pytest.mark.parametrize("heads, kv, dim, dtype, lens", [
    (32, 4, 128, torch.bfloat16, [1, 64, 65, 128, 0, 700, 4097, 5000, 2]), (3, 3, 64, torch.float32, [129, 192, 1, 1000]),
    (16, 1, 128, torch.float32, [1 + i % 70 for i in range(600)]), (34, 2, 64, torch.bfloat16, [100, 64, 1]),
    (4, 1, 64, torch.bfloat16, [1 + i * 37 % 65 for i in range(2500)]), (8, 4, 128, torch.bfloat16, [20000]),
    (8, 4, 128, torch.bfloat16, [64 * 40] * 48)])
def test_a_step_divided_once_for_its_layers(cuda, heads, kv, dim, dtype, lens):
    """Layers of one plan leave the cache and the answers, to the bit, that calls without one do: new
    tokens of any size, not finite, or nobody's (block 0); and both what a store before them leaves."""
    ours, want, stored = (Setup(cuda, lens, kv, dim, seed=7, layer=1) for _ in range(3))
    n, reqs = i64(lens, cuda), torch.arange(len(lens), device=cuda)
    loc = torch.cat([ours.rows(r, [max(m, 1) - 1]) for r, m in enumerate(lens)])
    loc[2::11] = 0
    gen = torch.Generator(device=cuda).manual_seed(3)
    for step in range(3):  # the same division three times over
        plan = fp4_decode_plan(ours.pool, ours.table, reqs, n) if step != 1 else plan
        for layer in (0, 1):  # layer 0: nothing there yet
            q = ours.queries(heads, dtype, 10 * step + layer)
            k, v = (torch.randn(len(lens), kv, dim, device=cuda, generator=gen) for _ in range(2))
            k[::3] *= 2.0 ** (3 * step)
            v[1::4] *= 2.0 ** (3 * step)
            k[5::13, 0, 3], v[7::17, kv - 1, 60] = float("nan"), float("inf")
            k, v = k.to(dtype), v.to(dtype)
            a = fp4_decode_attention(q, ours.pool, layer, ours.table, reqs, n, 0.1, new=(loc, k, v), plan=plan)
            b = fp4_decode_attention(q, want.pool, layer, want.table, reqs, n, 0.1, new=(loc, k, v))
            stored.pool.set_kv_buffer(layer, loc, k, v)
            c = fp4_decode_attention(q, stored.pool, layer, stored.table, reqs, n, 0.1)
            for other in (a, c):
                assert torch.equal(other.isnan(), b.isnan()) and torch.equal(other.nan_to_num(), b.nan_to_num())
            for x in ("k_codes", "v_codes", "k_scale", "v_scale"):
                assert torch.equal(getattr(ours.pool, x)[layer], getattr(want.pool, x)[layer]), x
                assert torch.equal(getattr(stored.pool, x)[layer], getattr(want.pool, x)[layer]), x
    ok = ~b.isnan().any(1).cpu()
    at = ok.nonzero()[:, 0].tolist()
    ours.check(a[ok.to(cuda)], q[ok.to(cuda)], 0.1, reqs=at, lens=[lens[i] for i in at])


def test_a_plan_of_other_lengths_answers_nothing_wrong(cuda):
    """Lengths and requests that change behind the plan: the right answer or NaN."""
    lens = [500, 64, 3000, 1, 200, 700]
    s = Setup(cuda, lens, 2, 128, spare=4)
    q, n, reqs = s.queries(8, torch.bfloat16), i64(lens, cuda), torch.arange(6, device=cuda)
    plan = fp4_decode_plan(s.pool, s.table, reqs, n)
    for m, r in [(n + 1, reqs), (n + 64, reqs), (n - 1, reqs), (n // 2, reqs), (n.flip(0), reqs), (n * 0, reqs), (n, reqs.flip(0))]:
        want = fp4_decode_attention(q, s.pool, s.layer, s.table, r, m, 0.1)
        got = fp4_decode_attention(q, s.pool, s.layer, s.table, r, m, 0.1, plan=plan)
        ok = got.isnan().all(1) | ((got.float() - want.float()).abs() <= 2**-7 * want.float().abs().amax(1, keepdim=True)).all(1)
        assert ok.all(), (m, r, ok)
    s.check(fp4_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1, plan=plan), q, 0.1)


def test_plans_and_pools_are_checked(cuda):
    s = Setup(cuda, [100, 100], 2, 64)
    q, r, n = s.queries(4, torch.bfloat16), torch.arange(2), i64([100, 100], cuda)
    plan = fp4_decode_plan(s.pool, s.table, r, n)
    more = fp4_decode_plan(s.pool, s.table, i64([0, 1, 0], cuda), n[:1].repeat(3))
    wider = fp4_decode_plan(Setup(cuda, [100, 100], 4, 64).pool, s.table, r, n)
    for bad in (more, wider, plan._replace(workspace=plan.workspace.cpu())):
        with pytest.raises(ValueError, match="plan"):
            fp4_decode_attention(q, s.pool, s.layer, s.table, r, n, 0.1, plan=bad)
    few = fp4_decode_plan(s.pool, s.table, r[:1], n[:1])
    assert fp4_decode_attention(q, s.pool, s.layer, s.table, r, n, 0.1, plan=few._replace(bs=2)).isnan().all()
    with pytest.raises(ValueError, match="Fp8TokenToKVPool"):
        fp8_decode_attention(q, s.pool, s.layer, s.table, r, n, 0.1)
    with pytest.raises(ValueError, match="Fp4TokenToKVPool"):
        fp4_decode_attention(q, Setup8(cuda, [100, 100], 2, 64).pool, s.layer, s.table, r, n, 0.1)
    for bad, said in ((dict(q=q[:, :3]), "divisible"), (dict(q=q.half()), "dtype"), (dict(q=q.cpu()), "lies on"),
                      (dict(table=s.table.long()), "int32"), (dict(n=i64([1, 2, 3], cuda)), "entries")):
        a = {**dict(q=q, table=s.table, n=n), **bad}
        with pytest.raises(ValueError, match=said):
            fp4_decode_attention(a["q"], s.pool, s.layer, a["table"], r, a["n"], 0.1)
    assert fp4_decode_attention(q[:0], s.pool, s.layer, s.table, r[:0], n[:0], 0.1).shape == (0, 256)


def test_replayed_graphs_with_growing_lengths(cuda):
    """Two captured calls of different shapes, replayed in turn while lengths change in place and other
    batches run eagerly between them."""
    lens = [500, 2000, 64]
    s = Setup(cuda, lens, 2, 128)
    qa, qb = s.queries(8, torch.bfloat16, 1), s.queries(2, torch.float32, 2)
    na, nb = i64([100, 1, 30], cuda), i64([64, 1000, 2], cuda)
    reqs = torch.arange(3, device=cuda)

    def a():
        return fp4_decode_attention(qa, s.pool, s.layer, s.table, reqs, na, 0.1)

    def b():
        return fp4_decode_attention(qb, s.pool, s.layer, s.table, reqs, nb, 0.1)

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
        fp4_decode_attention(s.queries(8, torch.bfloat16, 7), s.pool, s.layer, s.table, reqs, i64(lens, cuda), 0.1)
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
                outs.append(fp4_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, outs[i % 2])
    for i in range(2):
        s.check(outs[i], qs[i], 0.1)


def test_a_quest_plan_is_no_dense_plan(cuda):
    lens = [500, 64, 0, 1300]
    s = Setup(cuda, lens, 2, 128)
    q, reqs, n = s.queries(8, torch.bfloat16), torch.arange(4, device=cuda), i64(lens, cuda)
    quest = QuestAlgorithm(128, 64, cuda)
    quest.init_storage(0, 2, 4, s.table.shape[1] * 64, 2, 128)
    sparse = quest.decode_step_blocks(reqs, n, s.pool, s.table).plan
    with pytest.raises(ValueError, match="plan"):
        fp4_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1, plan=sparse)
    before = s.pool.k_codes.clone()
    new = (s.rows(0, [499] * 4), *(torch.randn(4, 2, 128, device=cuda) for _ in range(2)))
    out = fp4_decode_attention(q, s.pool, s.layer, s.table, reqs, n, 0.1, new=new, plan=sparse._replace(top_k=0))
    assert out.isnan().all() and torch.equal(before, s.pool.k_codes)
    assert of.BLOCK == o4.BLOCK
