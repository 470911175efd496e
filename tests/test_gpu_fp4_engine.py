"""The paged request pool, the 4-bit cache and the backends together, as an engine runs them: the engine's
tests of the 8-bit pool (tests/test_gpu_fp8_engine.py) over the 4-bit one and its definition, and a model's
layer from its QKV product on."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import fp4_cache as o4
from oracle import fp8_cache as of
from qwenquest_amd import QKNormRotary
from qwenquest_amd.attention import DenseBackend, QuestHiSparseBackend, QuestOnlyBackend
from qwenquest_amd.attention.ops import fp4_decode_attention, fp4_decode_plan, fp4_extend_attention
from qwenquest_amd.batch import ForwardBatch, ForwardMode
from qwenquest_amd.memory import ReqToTokenPool
from qwenquest_amd.paged import BlockReqToTokenPool, Fp4TokenToKVPool
from tests import test_gpu_fp8_engine as engine
from tests.test_gpu_fp8_engine import (  # noqa: F401 - collected here, over the 4-bit pool
    i64,
    test_a_divided_step_of_quest,
    test_a_prefill_cannot_be_traced,
    test_a_server_s_life,
    test_a_step_captured_apart_from_its_layers,
    test_a_step_s_division_stays_with_its_stream_and_capture,
    test_bounds_left_behind_select_nothing,
    test_decode_steps_in_a_replayed_graph,
    test_padded_entries_of_a_decode_batch,
    test_phases_are_the_step_in_two,
    test_prefills_without_tokens_and_with_rows_past_them,
    test_selections_in_wide_tables,
)

pytestmark = pytest.mark.gpu


def tolerance(out, spread, size, n, *args):
    """The 8-bit cache's, and what the prefill's f16 weights lose where the heaviest tokens' codes are 0 (tests/
    test_gpu_fp4_extend.py): n 1.5 2^-31 max(p |v|), of which every term is in the spread of some channel."""
    return of.attend_tolerance(out, spread, size, n, *args) + n * 1.5 * 2.0**-31 * spread.max(-1, keepdims=True)


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    monkeypatch.setattr(engine, "Fp8TokenToKVPool", Fp4TokenToKVPool)
    monkeypatch.setattr(engine, "of", SimpleNamespace(Cache=o4.Cache, attend=of.attend, attend_tolerance=tolerance))


def test_a_quest_step_refuses_another_step_s_plan(cuda):
    e = engine.Engine(cuda, "quest", 1, 16, 4, 128, torch.bfloat16, 2, 2000, 70, top_k=512)
    e.be.quest.trace = None
    e.prefill([0, 1], [700, 63])
    rpi, seq = i64([0, 1], cuda), i64([701, 64], cuda)
    loc, pos = e.rtp.assign_decode(rpi, seq)
    batch = ForwardBatch(ForwardMode.DECODE, None, pos, rpi, seq, loc, e.rtp, e.kvp, e.be)
    e.be.init_forward_metadata(batch)
    q, k, v = e.rand(2, 16, 128), e.rand(2, 4, 128), e.rand(2, 4, 128)
    step = e.be.quest._step
    plan, dense = step.plan, fp4_decode_plan(e.kvp, e.rtp.block_table, rpi, seq)
    for bad in (dense, plan._replace(bs=1), plan._replace(top_k=576), plan._replace(workspace=plan.workspace[256:])):
        step.plan = bad
        with pytest.raises(ValueError, match="plan"):
            e.be.forward(q, k, v, e.mods[0], batch)
    step.plan = dense._replace(top_k=512)  # does not show what it is of: no answer, and all of it written
    assert e.be.forward(q, k, v, e.mods[0], batch).isnan().all()
    step.plan = plan
    assert not e.be.forward(q, k, v, e.mods[0], batch).isnan().any()


def test_pools_that_do_not_go_together(cuda):
    paged, rows = BlockReqToTokenPool(2, 300, 9, cuda), ReqToTokenPool(2, 300, cuda)
    fp4 = Fp4TokenToKVPool(9, 1, 2, 128, cuda)
    cfg = {"algorithm": "quest", "top_k": 128, "quest_page_size": 64}
    with pytest.raises(ValueError, match="Fp4TokenToKVPool needs a BlockReqToTokenPool"):
        DenseBackend(rows, fp4)
    with pytest.raises(ValueError, match="blocks"):
        DenseBackend(BlockReqToTokenPool(2, 300, 10, cuda), fp4)
    with pytest.raises(ValueError, match="quest_page_size must be 64"):
        QuestOnlyBackend(paged, fp4, {**cfg, "quest_page_size": 32})
    with pytest.raises(ValueError, match="MHATokenToKVPool"):
        QuestHiSparseBackend(paged, fp4, cfg, host_pool_size=100)


def test_blocks_past_32_bit_offsets(cuda):
    """A layer of more than 2^32 bytes of codes: its last blocks written, read, bounded and attended."""
    kv, dim, blocks = 16, 128, 70_000  # 65536 bytes a block
    pool = Fp4TokenToKVPool(blocks, 1, kv, dim, cuda)
    assert pool.k_codes[0].numel() > 1 << 32
    ids = [blocks - 1, 1, blocks - 2, blocks // 2]
    table = torch.tensor([ids], dtype=torch.int32, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(0)
    loc = torch.tensor([b * 64 + t for b in ids for t in range(64)], device=cuda)
    k, v = (torch.empty((256, kv, dim), device=cuda).normal_(generator=gen).to(torch.bfloat16) for _ in range(2))
    pool.set_kv_buffer(0, loc, k, v)
    cache = o4.Cache(5, kv, dim)  # the same in small blocks
    cache.write(np.arange(64, 320), k.double().cpu().numpy(), v.double().cpu().numpy())
    kw, vw = cache.rows(np.arange(64, 320))
    got = pool.get_rows(0, loc, torch.float32)
    assert np.array_equal(got[0].cpu().numpy(), kw) and np.array_equal(got[1].cpu().numpy(), vw)
    q = torch.empty((2, 32, dim), device=cuda).normal_(generator=gen).to(torch.bfloat16)
    scale, n = dim**-0.5, 230
    for out, row, seen in (
            (fp4_decode_attention(q[:1], pool, 0, table, i64([0], cuda), i64([n], cuda), scale), q[0], n),
            (fp4_extend_attention(q, pool, 0, table, i64([0], cuda), i64([n], cuda), i64([n - 2], cuda), i64([2], cuda), scale)[1:], q[1], n)):
        want, spread, size = of.attend(row.double().cpu().numpy(), kw[:seen], vw[:seen], scale)
        tol = tolerance(want, spread, size, seen, dim, True, 12)
        assert (np.abs(out[0].double().cpu().numpy().reshape(want.shape) - want) <= tol).all()
    from qwenquest_amd.quest import QuestAlgorithm

    quest = QuestAlgorithm(128, 64, cuda)
    quest.init_storage(0, 1, 1, 256, kv, 64)
    with pytest.raises(ValueError, match="does not hold"):
        quest.update_prefill_representations_blocks(i64([0], cuda), i64([256], cuda), pool, table)


@pytest.mark.parametrize("backend", ["dense", "quest"])
def test_a_layer_from_its_qkv_product_on(cuda, backend):
    """Norms, rotation, the 4-bit cache and its attention in one run: chunked prefill and decode steps of two
    requests, every output against the formulas from the QKV product to the output in float64 - but that what the
    cache keeps is of the rotation's own bf16 keys, which the formulas' keys are within a rounding of."""
    heads, kv, dim = 16, 4, 128
    gen = torch.Generator(device=cuda).manual_seed(11)
    rtp, kvp = BlockReqToTokenPool(2, 900, 40, cuda), Fp4TokenToKVPool(40, 1, kv, dim, cuda)
    be = (DenseBackend(rtp, kvp) if backend == "dense" else
          QuestOnlyBackend(rtp, kvp, {"algorithm": "quest", "top_k": 512, "quest_page_size": 64}))
    wq, wk = (1 + 0.2 * torch.empty(dim, device=cuda).normal_(generator=gen) for _ in range(2))

    class Layer:
        layer_id, scaling = 0, dim**-0.5
        rotary = QKNormRotary(heads, kv, dim, q_weight=wq, k_weight=wk, base=1e6, device=cuda)

    cache, lens = o4.Cache(40, kv, dim), [0, 0]
    rpi = torch.arange(2, device=cuda)
    freq = 1e6 ** (-np.arange(64) / 64.0)

    def formula(x, w, pos):
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w.double().cpu().numpy()
        t = (pos[:, None] * freq)[:, None]
        a, b = y[..., :64], y[..., 64:]
        return np.concatenate([a * np.cos(t) - b * np.sin(t), b * np.cos(t) + a * np.sin(t)], -1)

    for new in ([300, 70], [64, 200], [1, 1], [1, 1], [150, 150], [1, 1], [1, 1]):
        n, decode = sum(new), sum(new) == 2
        pre, ext = i64(lens, cuda), i64(new, cuda)
        loc, pos = rtp.assign_decode(rpi, pre + 1) if decode else rtp.assign(rpi, pre, ext, n)
        batch = ForwardBatch(ForwardMode.DECODE if decode else ForwardMode.EXTEND, None, pos, rpi, pre + ext, loc, rtp, kvp, be,
                             extend_prefix_lens=pre, extend_seq_lens=ext)
        be.init_forward_metadata(batch)
        qkv = (torch.empty((n, (heads + 2 * kv) * dim), device=cuda).normal_(generator=gen) * 2).to(torch.bfloat16)
        out = be.forward_qkv(qkv, Layer, batch)
        be.on_extend_finished(batch)
        x, p = qkv.double().cpu().numpy().reshape(n, -1, dim), pos.cpu().numpy()
        q, k, v = Layer.rotary(qkv, pos)
        for got, want in ((q, formula(x[:, :heads], wq, p)), (k, formula(x[:, heads : heads + kv], wk, p))):
            pair = np.hypot(want[..., :64], want[..., 64:])
            err = np.abs(got.double().cpu().numpy() - want)
            assert (err <= 2.0**-8 * np.abs(want) + 2.0**-19 * np.concatenate([pair, pair], -1)).all()
        cache.write(loc.cpu().numpy(), k.double().cpu().numpy(), v.double().cpu().numpy())
        at = 0
        for r in range(2):
            for t in sorted({0, new[r] // 2, new[r] - 1}):
                s = lens[r] + t + 1
                if decode and backend == "quest" and s > 512:
                    seen = be._positions[r].cpu().numpy()
                else:
                    seen = np.arange(s)
                kw, vw = cache.rows(rtp.req_to_token[r].cpu().numpy()[seen])
                want, spread, size = of.attend(q[at + t].double().cpu().numpy(), kw, vw, Layer.scaling)
                tol = tolerance(want, spread, size, len(seen), dim, True, 12)
                assert (np.abs(out[at + t].double().cpu().numpy().reshape(want.shape) - want) <= tol).all()
            at += new[r]
        lens = [a + b for a, b in zip(lens, new)]
    assert max(lens) > 512
    rtp.check_errors()


@pytest.mark.parametrize("kv, group, lens, top_k", [
    (1, 8, [700 + 13 * i for i in range(256)], 512), (1, 16, [700] * 257, 512), (1, 1, [3000], 2112), (1, 5, [2600, 1, 2112, 2113, 64] * 20, 2112),
    (2, 7, [600 + 5 * i for i in range(128)], 512), (2, 16, [5000, 100], 2112), (3, 4, [900 + 50 * i for i in range(85)], 832),
    (8, 8, [1300, 40, 1024, 1025] * 8, 1024), (8, 2, [4000] * 3, 2176), (8, 4, [9000], 2624), (4, 8, [9000], 2688), (16, 4, [800] * 16, 576),
    (64, 1, [700, 650, 600, 30], 512)])
def test_a_divided_step_of_quest_with_any_number_of_kv_heads(cuda, kv, group, lens, top_k):
    """As many requests as a slice may meet, selections up to the most that the attention makes itself and past it:
    positions, cache and answers, to the bit, of the step whose selection is a launch of its own."""
    dim, bs, width = 128, len(lens), max(lens) + 3
    gen = torch.Generator(device=cuda).manual_seed(kv * bs)
    rtp = BlockReqToTokenPool(bs, width, sum(n // 64 + 2 for n in lens) + 2, cuda)
    kvp = Fp4TokenToKVPool(rtp.num_blocks, 1, kv, dim, cuda)
    be = QuestOnlyBackend(rtp, kvp, {"algorithm": "quest", "top_k": top_k, "quest_page_size": 64})
    reqs, had = torch.arange(bs, device=cuda), [n - 1 for n in lens]
    total = sum(had)
    loc, _ = rtp.assign(reqs, i64([0] * bs, cuda), i64(had, cuda), total)
    pages = torch.randn(total // 64 + 1, kv, dim, device=cuda, generator=gen).repeat_interleave(64, 0)[:total]
    kvp.set_kv_buffer(0, loc, pages + torch.randn(total, kv, dim, device=cuda, generator=gen),
                      torch.randn(total, kv, dim, device=cuda, generator=gen))
    be.quest.update_prefill_representations_blocks(reqs, i64(had, cuda), kvp, rtp.block_table)
    seq = i64(lens, cuda)
    for step in range(2):
        loc, pos = rtp.assign_decode(reqs, seq)
        batch = ForwardBatch(ForwardMode.DECODE, None, pos, reqs, seq, loc, rtp, kvp, be)
        q, k, v = (torch.randn(bs, h, dim, device=cuda, generator=gen).bfloat16() for h in (group * kv, kv, kv))
        if kv * dim > 1024:  # more channels than page scores are taken of
            be.init_forward_metadata(batch)
            with pytest.raises(ValueError, match="exceeds 1024"):
                be.forward(q, k, v, engine.Layer(0, dim), batch)
            return
        if step:
            q[:] = 0  # every page scores alike
        be.init_forward_metadata(batch)
        got = []
        for planned in (True, False):
            if not planned:
                be.quest._step.plan = None
            be._positions.fill_(-7)
            out = be.forward(q, k, v, engine.Layer(0, dim), batch)
            got.append([t.clone() for t in (out, be._positions, kvp.k_codes, kvp.v_codes, kvp.k_scale, kvp.v_scale)])
        assert not got[0][0].isnan().any()
        assert all(torch.equal(a, b) for a, b in zip(*got))
        seq = seq + 1
    rtp.check_errors()
