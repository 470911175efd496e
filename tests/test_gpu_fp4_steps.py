"""Steps over the pools of codes as a backend does not make them: a Quest step with another step's plan, operators
under torch.jit.trace."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from qwenquest_amd import QKNormRotary
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
