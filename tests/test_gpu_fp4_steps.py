"""Steps over the 4-bit pool that go wrong or go through the functions of one kind of pool: a Quest step with another
step's plan, the functions by their pools, operators under torch.jit.trace."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from qwenquest_amd import QKNormRotary, QuestAlgorithm
from qwenquest_amd.attention import ops
from qwenquest_amd.batch import ForwardBatch, ForwardMode
from qwenquest_amd.paged import Fp4TokenToKVPool, Fp8TokenToKVPool
from tests import test_gpu_fp8_engine as engine
from tests.test_gpu_fp8_engine import i64

pytestmark = pytest.mark.gpu

CACHE = ("k_codes", "v_codes", "k_scale", "v_scale")


def quest_step(monkeypatch, cuda, kind, had, top_k=512, heads=16, kv=4):
    monkeypatch.setattr(engine, "Fp8TokenToKVPool", kind)
    e = engine.Engine(cuda, "quest", 1, heads, kv, 128, torch.bfloat16, len(had), 2000, 30 * len(had) + 10, top_k=top_k)
    e.be.quest.trace = None
    reqs = list(range(len(had)))
    rpi, pre, ext = i64(reqs, cuda), i64([0] * len(had), cuda), i64(had, cuda)
    loc, pos = e.rtp.assign(rpi, pre, ext, sum(had))
    e.kvp.set_kv_buffer(0, loc, e.rand(sum(had), kv, 128), e.rand(sum(had), kv, 128))
    e.be.quest.update_prefill_representations_blocks(rpi, ext, e.kvp, e.rtp.block_table)
    seq = ext + 1
    loc, pos = e.rtp.assign_decode(rpi, seq)
    batch = ForwardBatch(ForwardMode.DECODE, None, pos, rpi, seq, loc, e.rtp, e.kvp, e.be)
    e.be.init_forward_metadata(batch)
    return e, batch, [e.rand(len(had), h, 128) for h in (heads, kv, kv)]


@pytest.mark.parametrize("kind, kv, had", [(Fp8TokenToKVPool, 4, [700, 63]), (Fp4TokenToKVPool, 4, [700, 63]),
                                           (Fp4TokenToKVPool, 1, [600, 64, 900, 1, 127] * 9), (Fp4TokenToKVPool, 8, [1300] * 20)])
def test_a_quest_step_with_another_plan_keeps_its_tokens(monkeypatch, cuda, kind, kv, had):
    """No answer to any request, but the new tokens are in the cache as a step of its own plan leaves them there, and no
    other row is touched."""
    e, batch, (q, k, v) = quest_step(monkeypatch, cuda, kind, had, heads=4 * kv, kv=kv)
    before = [getattr(e.kvp, x).clone() for x in CACHE]
    dense = ops.coded_decode_plan(e.kvp, e.rtp.block_table, batch.req_pool_indices, batch.seq_lens)
    plan = e.be.quest._step.plan
    e.be.quest._step.plan = dense._replace(top_k=512)  # does not show what it is of
    assert e.be.forward(q, k, v, e.mods[0], batch).isnan().all()
    got = [getattr(e.kvp, x).clone() for x in CACHE]
    for x, old in zip(CACHE, before):
        getattr(e.kvp, x).copy_(old)
    e.kvp.set_kv_buffer(0, batch.out_cache_loc, k, v)
    assert all(torch.equal(getattr(e.kvp, x), y) for x, y in zip(CACHE, got))
    assert not all(torch.equal(x, y) for x, y in zip(before, got))
    e.be.quest._step.plan = plan
    assert not e.be.forward(q, k, v, e.mods[0], batch).isnan().any()


def test_quest_steps_by_their_kind_of_pool(monkeypatch, cuda):
    """fp8_quest_step and fp4_quest_step are the backend's step, and refuse the other pool."""
    for kind, own, other in ((Fp8TokenToKVPool, ops.fp8_quest_step, ops.fp4_quest_step), (Fp4TokenToKVPool, ops.fp4_quest_step, ops.fp8_quest_step)):
        e, b, (q, k, v) = quest_step(monkeypatch, cuda, kind, [700, 63])
        want = e.be.forward(q, k, v, e.mods[0], b)
        pos = torch.empty_like(e.be._positions)
        args = (q, k, v, b.out_cache_loc, e.kvp, 0, e.rtp.block_table, e.be.quest, b.req_pool_indices, pos, e.mods[0].scaling)
        assert torch.equal(own(*args), want) and torch.equal(pos[:2], e.be._positions[:2])
        with pytest.raises(ValueError, match="TokenToKVPool"):
            other(*args)


def test_a_pool_that_names_no_kind_holds_8_bit_blocks(cuda):
    """Any object with an 8-bit pool's attributes serves the 8-bit functions."""
    pool = Fp8TokenToKVPool(6, 1, 2, 128, cuda)
    gen = torch.Generator(device=cuda).manual_seed(0)
    rand = lambda *shape: torch.empty(shape, device=cuda).normal_(generator=gen).bfloat16()  # noqa: E731
    pool.set_kv_buffer(0, torch.arange(64, 364, device=cuda), rand(300, 2, 128), rand(300, 2, 128))
    plain = SimpleNamespace(**{x: getattr(pool, x) for x in ("device", "num_blocks", "kv_heads", "head_dim", "num_layers", "k_codes", "k_scale",
                                                             "layer_args", "new_rows")})
    table, rpi, n = torch.arange(1, 6, dtype=torch.int32, device=cuda)[None], i64([0], cuda), i64([290], cuda)
    q = rand(1, 8, 128)
    want = ops.fp8_decode_attention(q, pool, 0, table, rpi, n, 0.1)
    plan = ops.fp8_decode_plan(plain, table, rpi, n)
    assert torch.equal(ops.fp8_decode_attention(q, plain, 0, table, rpi, n, 0.1), want)
    assert torch.equal(ops.fp8_decode_attention(q, plain, 0, table, rpi, n, 0.1, plan=plan), want)
    q = rand(20, 8, 128)
    assert torch.equal(*(ops.fp8_extend_attention(q, p, 0, table, rpi, n, n - 20, i64([20], cuda), 0.1) for p in (pool, plain)))
    quests = []
    for p in (pool, plain):
        quest = QuestAlgorithm(128, 64, cuda)
        quest.init_storage(0, 1, 1, 320, 2, 128)
        quest.update_prefill_representations_blocks(rpi, n, p, table)
        quest.decode_step_blocks(rpi, n, p, table)
        quests.append(quest)
    assert torch.equal(quests[0].page_k_bounds[0, 0, :4], quests[1].page_k_bounds[0, 0, :4])
    args = (q[:1], rand(1, 2, 128), rand(1, 2, 128), i64([64 + 289], cuda))
    outs = [ops.fp8_quest_step(*args, p, 0, table, x, rpi, torch.empty((1, 128), dtype=torch.int32, device=cuda), 0.1) for p, x in zip((pool, plain), quests)]
    assert torch.equal(*outs)
    with pytest.raises(ValueError, match="Fp4TokenToKVPool"):
        ops.fp4_decode_attention(q[:1], plain, 0, table, rpi, n, 0.1)


def test_operators_that_a_trace_would_lose_refuse_it(monkeypatch, cuda):
    op = QKNormRotary(4, 2, 64, device=cuda)
    x, pos = torch.randn(5, 512, device=cuda), torch.arange(5, device=cuda)

    def refused(f, *args):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, args, check_trace=False)

    refused(lambda x: op(x, pos), x)
    refused(lambda x: op.apply(x[:, :256], x[:, 256:384], pos), x)
    for kind in (Fp4TokenToKVPool, Fp8TokenToKVPool):
        e, b, (q, k, v) = quest_step(monkeypatch, cuda, kind, [700, 63])
        before = e.kvp.k_codes.clone()
        table, rpi, n = e.rtp.block_table, b.req_pool_indices, b.seq_lens
        refused(lambda loc: e.kvp.get_rows(0, loc), b.out_cache_loc)
        refused(lambda k: (e.kvp.set_kv_buffer(0, b.out_cache_loc, k, v), k)[1], k)
        refused(lambda q: ops.coded_decode_attention(q, e.kvp, 0, table, rpi, n, 0.1), q)
        refused(lambda n: ops.coded_decode_plan(e.kvp, table, rpi, n).workspace, n)
        refused(lambda q: ops.coded_extend_attention(q, e.kvp, 0, table, rpi, n, n - 1, n * 0 + 1, 0.1), q)
        refused(lambda q: e.be.forward(q, k, v, e.mods[0], b), q)
        refused(lambda n: e.be.quest.decode_step_blocks(rpi, n, e.kvp, table).seq_lens, n)
        refused(lambda n: (e.be.quest.update_prefill_representations_blocks(rpi, n, e.kvp, table), n)[1], n)
        dense = engine.DenseBackend(e.rtp, e.kvp)
        refused(lambda q: dense.forward(q, k, v, e.mods[0], b), q)
        layer = SimpleNamespace(layer_id=0, scaling=0.1, rotary=QKNormRotary(16, 4, 128, device=cuda))
        refused(lambda x: dense.forward_qkv(x, layer, b), torch.randn(2, 24 * 128, device=cuda).bfloat16())
        assert torch.equal(before, e.kvp.k_codes)
        assert not e.be.forward(q, k, v, e.mods[0], b).isnan().any()
