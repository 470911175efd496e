"""The paged request pool, the 8-bit cache and the backends together, as an engine runs them: admission,
chunked prefill, decode steps, requests that finish and slots that are used again - against the
cache and the attention by their definitions on the host."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import bf16
from oracle import fp8_cache as of
from oracle import quest as oq
from qwenquest_amd.attention import DenseBackend, QuestHiSparseBackend, QuestOnlyBackend
from qwenquest_amd.batch import ForwardBatch, ForwardMode
from qwenquest_amd.memory import MHATokenToKVPool, ReqToTokenPool
from qwenquest_amd.paged import BlockReqToTokenPool, Fp8TokenToKVPool
from qwenquest_amd.quest import QuestTrace

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, layer_id, dim):
        self.layer_id, self.scaling = layer_id, dim**-0.5


def i64(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int64).to(dev)


class Engine:
    """What an engine keeps, and the same on the host: tokens of each request per layer."""

    def __init__(self, dev, backend, layers, heads, kv, dim, dtype, reqs, width, blocks, top_k=256, avoid=False, seed=0):
        self.dev, self.layers, self.heads, self.kv, self.dim, self.dtype = dev, layers, heads, kv, dim, dtype
        self.rtp = BlockReqToTokenPool(reqs, width, blocks, dev)
        self.kvp = Fp8TokenToKVPool(blocks, layers, kv, dim, dev)
        self.top_k = top_k
        if backend == "quest":
            self.be = QuestOnlyBackend(self.rtp, self.kvp, {"algorithm": "quest", "top_k": top_k, "quest_page_size": 64,
                                                            "avoid_recent_overlap": avoid})
            self.be.quest.trace = QuestTrace()
        else:
            self.be = DenseBackend(self.rtp, self.kvp)
        self.avoid = avoid
        self.gen = torch.Generator(device=dev).manual_seed(seed)
        self.cache = [of.Cache(blocks, kv, dim) for _ in range(layers)]
        self.lens = {}
        self.mods = [Layer(i, dim) for i in range(layers)]

    def rand(self, *shape):
        return torch.empty(shape, device=self.dev).normal_(generator=self.gen).to(self.dtype)

    def check(self, out, q, ks, scale=None):
        k, v = ks
        qn = q.double().cpu().numpy()
        want, spread, size = of.attend(qn, k, v, self.dim**-0.5)
        bf = self.dtype == torch.bfloat16
        # 12 bits of a weight cover the prefill's rounding as well as the decode's
        tol = of.attend_tolerance(want, spread, size, len(k), self.dim, bf, 12 if bf else 22)
        err = np.abs(out.double().cpu().numpy().reshape(want.shape) - want)
        assert (err <= tol).all(), (err / tol).max()

    def prefill(self, reqs, new):
        prefix = [self.lens.get(r, 0) for r in reqs]
        rpi, pre, ext = i64(reqs, self.dev), i64(prefix, self.dev), i64(new, self.dev)
        n = sum(new)
        loc, pos = self.rtp.assign(rpi, pre, ext, n)
        batch = ForwardBatch(ForwardMode.EXTEND, None, pos, rpi, pre + ext, loc, self.rtp, self.kvp, self.be,
                             extend_prefix_lens=pre, extend_seq_lens=ext)
        self.be.init_forward_metadata(batch)
        for layer in self.mods:
            q, k, v = self.rand(n, self.heads, self.dim), self.rand(n, self.kv, self.dim) * 2, self.rand(n, self.kv, self.dim)
            out = self.be.forward(q, k, v, layer, batch)
            assert out.shape == (n, self.heads * self.dim) and out.dtype == q.dtype
            self.cache[layer.layer_id].write(loc.cpu().numpy(), k.float().cpu().numpy(), v.float().cpu().numpy())
            at = 0
            for r, p, m in zip(reqs, prefix, new):
                for t in sorted({0, m // 2, m - 1}) if m else []:
                    self.check(out[at + t], q[at + t], self.cache[layer.layer_id].rows(self.rows(r, p + t + 1)))
                at += m
        self.be.on_extend_finished(batch)
        for r, p, m in zip(reqs, prefix, new):
            self.lens[r] = p + m

    def rows(self, r, n):
        return self.rtp.req_to_token[r, :n].long().cpu().numpy()

    def decode(self, reqs):
        """One eager step of these requests; the attended positions come from the definition."""
        seq = [self.lens[r] + 1 for r in reqs]
        rpi, sl = i64(reqs, self.dev), i64(seq, self.dev)
        loc, pos = self.rtp.assign_decode(rpi, sl)
        batch = ForwardBatch(ForwardMode.DECODE, None, pos, rpi, sl, loc, self.rtp, self.kvp, self.be)
        bounds = [self.bounds(layer, reqs, seq) for layer in range(self.layers)]
        self.be.init_forward_metadata(batch)
        for layer in self.mods:
            q, k, v = self.rand(len(reqs), self.heads, self.dim), self.rand(len(reqs), self.kv, self.dim), self.rand(len(reqs), self.kv, self.dim)
            out = self.be.forward(q, k, v, layer, batch)
            c = self.cache[layer.layer_id]
            c.write(loc.cpu().numpy(), k.float().cpu().numpy(), v.float().cpu().numpy())
            for i, (r, s) in enumerate(zip(reqs, seq)):
                at = np.arange(s)
                if isinstance(self.be, QuestOnlyBackend):
                    at = self.selected(q[i], bounds[layer.layer_id][i], s)
                    got = self.be.quest.trace.records[-len(reqs) + i]
                    assert got.layer_id == layer.layer_id and got.positions.tolist() == at.tolist()
                self.check(out[i], q[i], c.rows(self.rows(r, s)[at]))
        for r, s in zip(reqs, seq):
            self.lens[r] = s

    def bounds(self, layer, reqs, seq):
        """Bounds of the pages that are complete before the step's own token, bf16 bits."""
        out = []
        for r, s in zip(reqs, seq):
            full = (s - 1) // 64
            k = self.cache[layer].rows(self.rows(r, full * 64))[0].reshape(full, 64, self.kv, self.dim)
            lo, hi = (bf16.from_f32(x.astype(np.float32)) for x in (k.min(1), k.max(1))) if full else (np.zeros((0, self.kv, self.dim), np.uint16),) * 2
            out.append(np.stack([lo, hi], -1))
        return out

    def selected(self, q, bounds, s):
        if s <= self.top_k:
            return np.arange(s)
        qbar = oq.group_queries(q.float().cpu().numpy()[None], self.kv, self.dim, self.dtype == torch.bfloat16)
        scores = oq.page_scores(qbar, bounds[None])[0]
        limit = s // 64 - 1 if self.avoid else s // 64
        pages = oq.topk_pages(scores, min(limit, len(scores)), self.top_k // 64 - 1)
        return np.concatenate([(pages[:, None] * 64 + np.arange(64)).reshape(-1), np.arange(s - 64, s)])

    def finish(self, r):
        self.be.on_request_finished(r)
        self.rtp.release(i64([r], self.dev))
        del self.lens[r]


@pytest.mark.parametrize("backend, heads, kv, dim, dtype, avoid", [
    ("quest", 16, 4, 128, torch.bfloat16, False), ("quest", 6, 2, 128, torch.bfloat16, True),
    ("quest", 8, 2, 64, torch.float32, False), ("dense", 10, 2, 128, torch.bfloat16, False), ("dense", 3, 3, 64, torch.float32, False)])
def test_a_server_s_life(cuda, backend, heads, kv, dim, dtype, avoid):
    e = Engine(cuda, backend, 2, heads, kv, dim, dtype, 4, 900, 50, avoid=avoid)
    e.prefill([2, 0], [300, 40])
    for _ in range(3):
        e.decode([0, 2])
    e.prefill([2, 3], [250, 64])  # a second chunk, and another request
    for i in range(70):
        e.decode([3, 2, 0] if i % 2 else [2, 3])
    e.finish(2)
    e.prefill([2], [500])  # the slot again, over blocks that were used
    for _ in range(4):
        e.decode([2, 0])
    e.rtp.check_errors()


def test_decode_steps_in_a_replayed_graph(cuda):
    """A captured step of every layer, replayed as lengths grow in place; eager steps between."""
    e, w = (Engine(cuda, "quest", 2, 8, 2, 128, torch.bfloat16, 3, 900, 50, seed=5) for _ in range(2))
    for x in (e, w):
        x.be.quest.trace = None
        x.prefill([0, 1, 2], [400, 63, 255])
    rpi, seq = torch.arange(3, device=cuda), i64([401, 64, 256], cuda)
    q, k, v = (torch.zeros(2, 3, h, 128, device=cuda, dtype=torch.bfloat16) for h in (8, 2, 2))

    def step(x):
        loc, pos = x.rtp.assign_decode(rpi, seq)
        batch = ForwardBatch(ForwardMode.DECODE, None, pos, rpi, seq, loc, x.rtp, x.kvp, x.be)
        x.be.init_forward_metadata(batch)
        return [x.be.forward(q[i], k[i], v[i], x.mods[i], batch) for i in range(2)]

    for t in (q, k, v):
        t.normal_(generator=e.gen)
    step(e), step(w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(e)
    for _ in range(6):
        seq += 1
        for t in (q, k, v):
            t.normal_(generator=e.gen)
        graph.replay()
        want = step(w)
        assert all(torch.equal(a, b) and not a.isnan().any() for a, b in zip(outs, want))
        assert torch.equal(e.kvp.k_codes, w.kvp.k_codes) and torch.equal(e.be.quest.page_k_bounds, w.be.quest.page_k_bounds)
    e.rtp.poll_errors()


@pytest.mark.parametrize("backend", ["dense", "quest"])
def test_a_step_s_division_stays_with_its_stream_and_capture(cuda, backend):
    """Layers on another stream, layers captured without their init_forward_metadata and replayed as
    lengths grow (dense), eager layers behind a capture that never ran, a part of the batch."""
    from dataclasses import replace

    e, w = (Engine(cuda, backend, 1, 32, 4, 128, torch.bfloat16, 3, 5000, 100, top_k=512, seed=5) for _ in range(2))
    for x in (e, w):
        if backend == "quest":
            x.be.quest.trace = None
        x.prefill([0, 1, 2], [700, 63, 2000])
    rpi, seq = torch.arange(3, device=cuda), i64([701, 64, 2001], cuda)
    q, k, v = (torch.zeros(3, h, 128, device=cuda, dtype=torch.bfloat16) for h in (32, 4, 4))

    def begin(x):
        loc, pos = x.rtp.assign_decode(rpi, seq)
        batch = ForwardBatch(ForwardMode.DECODE, None, pos, rpi, seq, loc, x.rtp, x.kvp, x.be)
        x.be.init_forward_metadata(batch)
        return batch

    def layer(x, batch):
        return x.be.forward(q, k, v, x.mods[0], batch)

    def same(out):
        want = layer(w, begin(w))
        assert not want.isnan().any() and torch.allclose(out.float(), want.float(), rtol=2**-7, atol=2**-9)
        assert torch.equal(e.kvp.k_codes, w.kvp.k_codes) and torch.equal(e.kvp.v_scale, w.kvp.v_scale)

    def more():
        seq.add_(1)
        for t in (q, k, v):
            t.normal_(generator=e.gen)

    more()
    side, batch = torch.cuda.Stream(), begin(e)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = layer(e, batch)
    torch.cuda.current_stream().wait_stream(side)
    same(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(e, batch)
    for _ in range(3 if backend == "dense" else 0):
        more()
        loc, _ = e.rtp.assign_decode(rpi, seq)
        batch.out_cache_loc.copy_(loc)
        e.be.init_forward_metadata(batch)
        graph.replay()
        same(out)
    more()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        captured = begin(e)
        layer(e, captured)
    e.rtp.assign_decode(rpi, seq)
    eager = begin(e)
    if backend == "dense":  # (Quest's layout of the capture has no values yet)
        eager.decode_plan = captured.decode_plan
        part = replace(eager, decode_plan=begin(e).decode_plan, req_pool_indices=rpi[:2], seq_lens=seq[:2],
                       out_cache_loc=eager.out_cache_loc[:2])
        whole = layer(e, eager)
        assert torch.allclose(e.be.forward(q[:2], k[:2], v[:2], e.mods[0], part).float(), whole[:2].float(), rtol=2**-7, atol=2**-9)
    else:
        e.be.quest._step.plan = e.be.quest._step.plan._replace(captured=True)
    same(layer(e, eager))


@pytest.mark.parametrize("backend", ["dense", "quest"])
def test_a_step_captured_apart_from_its_layers(cuda, backend):
    """init_forward_metadata in one graph, the layers in another: both are captured on the same stream,
    and the layers do not rely on memory of the first graph that a plan would lie in."""
    e, w = (Engine(cuda, backend, 1, 32, 4, 128, torch.bfloat16, 3, 5000, 100, top_k=512, seed=9) for _ in range(2))
    for x in (e, w):
        if backend == "quest":
            x.be.quest.trace = None
        x.prefill([0, 1, 2], [700, 63, 2000])
    rpi, seq = torch.arange(3, device=cuda), i64([701, 64, 2001], cuda)
    loc = torch.zeros(3, dtype=torch.int64, device=cuda)
    q, k, v = (torch.zeros(3, h, 128, device=cuda, dtype=torch.bfloat16) for h in (32, 4, 4))

    def batch_of(x, rows):
        return ForwardBatch(ForwardMode.DECODE, None, None, rpi, seq, rows, x.rtp, x.kvp, x.be)

    batch = batch_of(e, loc)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        e.be.init_forward_metadata(batch)
    plan = batch.decode_plan if backend == "dense" else e.be.quest._step.plan
    assert plan.captured > 0 and not plan.usable(plan.stream)
    with torch.cuda.graph(graphs[1]):
        stream = torch.cuda.current_stream().cuda_stream
        assert stream == plan.stream and not plan.usable(stream)
        out = e.be.forward(q, k, v, e.mods[0], batch)
    plan.workspace.fill_(255)  # nothing reads it
    for step in range(4):
        if step:
            seq.add_(1)
        for t in (q, k, v):
            t.normal_(generator=e.gen)
        loc.copy_(e.rtp.assign_decode(rpi, seq)[0])
        if backend == "quest" or step % 2:  # (Quest's layout comes from the first graph)
            graphs[0].replay()
            plan.workspace.fill_(255)
        graphs[1].replay()
        rows, _ = w.rtp.assign_decode(rpi, seq)
        other = batch_of(w, rows)
        w.be.init_forward_metadata(other)
        want = w.be.forward(q, k, v, w.mods[0], other)
        assert not want.isnan().any() and torch.equal(out, want)
        assert torch.equal(e.kvp.k_codes, w.kvp.k_codes) and torch.equal(e.kvp.v_scale, w.kvp.v_scale)


def test_a_quest_step_refuses_another_step_s_plan(cuda):
    from qwenquest_amd.attention.ops import fp8_decode_plan

    e = Engine(cuda, "quest", 1, 16, 4, 128, torch.bfloat16, 2, 2000, 70, top_k=512)
    e.be.quest.trace = None
    e.prefill([0, 1], [700, 63])
    rpi, seq = i64([0, 1], cuda), i64([701, 64], cuda)
    loc, pos = e.rtp.assign_decode(rpi, seq)
    batch = ForwardBatch(ForwardMode.DECODE, None, pos, rpi, seq, loc, e.rtp, e.kvp, e.be)
    e.be.init_forward_metadata(batch)
    q, k, v = e.rand(2, 16, 128), e.rand(2, 4, 128), e.rand(2, 4, 128)
    step = e.be.quest._step
    plan, dense = step.plan, fp8_decode_plan(e.kvp, e.rtp.block_table, rpi, seq)
    for bad in (dense, plan._replace(bs=1), plan._replace(top_k=576), plan._replace(workspace=plan.workspace[256:])):
        step.plan = bad
        with pytest.raises(ValueError, match="plan"):
            e.be.forward(q, k, v, e.mods[0], batch)
    step.plan = dense._replace(top_k=512)  # does not show what it is of: no answer, and all of it written
    assert e.be.forward(q, k, v, e.mods[0], batch).isnan().all()
    step.plan = plan
    assert not e.be.forward(q, k, v, e.mods[0], batch).isnan().any()


def test_padded_entries_of_a_decode_batch(cuda):
    """seq_lens 0: no row, no token stored, an output of zeros."""
    e = Engine(cuda, "dense", 1, 4, 2, 128, torch.bfloat16, 3, 300, 20)
    e.prefill([0, 1], [100, 30])
    rpi, seq = i64([0, 0, 1], cuda), i64([101, 0, 31], cuda)
    loc, pos = e.rtp.assign_decode(rpi, seq)
    assert loc[1] == 0
    batch = ForwardBatch(ForwardMode.DECODE, None, pos, rpi, seq, loc, e.rtp, e.kvp, e.be)
    q, k, v = e.rand(3, 4, 128), e.rand(3, 2, 128), e.rand(3, 2, 128)
    out = e.be.forward(q, k, v, e.mods[0], batch)
    e.cache[0].write(loc.cpu().numpy(), k.float().cpu().numpy(), v.float().cpu().numpy())
    for i in (0, 2):
        e.check(out[i], q[i], e.cache[0].rows(e.rows(int(rpi[i]), int(seq[i]))))
    assert not out[1].any() and not e.kvp.k_codes[0, 0].any()


@pytest.mark.parametrize("how", ["rolled back", "slot used again"])
def test_bounds_left_behind_select_nothing(cuda, how):
    """A request that is rolled back past a page's end and decodes other tokens, and one in a slot whose
    blocks went back without on_request_finished: the page that the step completes has no bounds
    yet, whatever stands in its place, and the selections are those of an engine without a past."""
    e, w = (Engine(cuda, "quest", 1, 16, 4, 128, torch.bfloat16, 2, 1000, 40, top_k=256, seed=4) for _ in range(2))
    gen = torch.Generator(device=cuda).manual_seed(8)
    prompt = [torch.randn(500, h, 128, device=cuda, generator=gen).bfloat16() for h in (16, 4, 4)]

    def run(x, mode, seq, q, k, v):
        n = q.shape[0]
        rpi, sl, pre = i64([1], cuda), i64([seq], cuda), i64([seq - n], cuda)
        ext = i64([n], cuda)
        loc, pos = x.rtp.assign(rpi, pre, ext, n) if mode is ForwardMode.EXTEND else x.rtp.assign_decode(rpi, sl)
        batch = ForwardBatch(mode, None, pos, rpi, sl, loc, x.rtp, x.kvp, x.be, extend_prefix_lens=pre, extend_seq_lens=ext)
        x.be.init_forward_metadata(batch)
        return x.be.forward(q, k, v, x.mods[0], batch)

    def token(size=1.0):
        return [torch.randn(1, h, 128, device=cuda, generator=gen).bfloat16() * size for h in (16, 4, 4)]

    run(e, ForwardMode.EXTEND, 500, *prompt)
    for seq in range(501, 516):  # large keys in page 7, which 513 finds complete
        run(e, ForwardMode.DECODE, seq, *token(30.0))
    if how == "slot used again":
        e.rtp.release(i64([1], cuda))
        run(e, ForwardMode.EXTEND, 500, *prompt)
    run(w, ForwardMode.EXTEND, 500, *prompt)
    # what was rolled back has left page 7 a larger scale, which its bounds show from 513 on
    for seq in range(501, 513 if how == "rolled back" else 516):
        q, k, v = token()
        a, b = (run(x, ForwardMode.DECODE, seq, q, k, v) for x in (e, w))
        got, want = (x.be.quest.trace.records[-1].positions.tolist() for x in (e, w))
        assert got == want, seq
        if how == "slot used again":
            assert torch.equal(a, b), seq


def prefill_batch(e, reqs, prefix, new):
    rpi, pre, ext = i64(reqs, e.dev), i64(prefix, e.dev), i64(new, e.dev)
    loc, pos = e.rtp.assign(rpi, pre, ext, sum(new))
    return ForwardBatch(ForwardMode.EXTEND, None, pos, rpi, pre + ext, loc, e.rtp, e.kvp, e.be, extend_prefix_lens=pre,
                        extend_seq_lens=ext)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("backend", ["dense", "quest"])
def test_prefills_without_tokens_and_with_rows_past_them(cuda, backend, dtype):
    """Both query types answer alike: as many rows as q has, NaN past the requests' tokens; a batch, and a
    decode batch, of nothing."""
    e = Engine(cuda, backend, 1, 4, 2, 64, dtype, 3, 300, 20, top_k=128)
    b = prefill_batch(e, [0, 1], [0, 0], [70, 5])
    q, k, v = e.rand(80, 4, 64), e.rand(75, 2, 64), e.rand(75, 2, 64)
    out = e.be.forward(q, k, v, e.mods[0], b)
    assert out.shape == (80, 256) and out.dtype == dtype and out[75:].isnan().all() and not out[:75].isnan().any()
    assert torch.equal(out[:75], e.be.forward(q[:75], k, v, e.mods[0], b))
    for shape in ((0, 4, 64), (0, 256)):
        b = prefill_batch(e, [0, 1], [70, 5], [0, 0])
        assert e.be.forward(e.rand(*shape), k[:0], v[:0], e.mods[0], b).shape == (0, 256)
        none = i64([], cuda)
        b = ForwardBatch(ForwardMode.DECODE, None, none, none, none, none, e.rtp, e.kvp, e.be)
        e.be.init_forward_metadata(b)
        assert e.be.forward(e.rand(*shape), k[:0], v[:0], e.mods[0], b).shape == (0, 256)
    e.rtp.check_errors()


def test_a_prefill_cannot_be_traced(cuda):
    e = Engine(cuda, "dense", 1, 4, 2, 128, torch.bfloat16, 1, 300, 10)
    b = prefill_batch(e, [0], [0], [20])
    q, k, v = e.rand(20, 4, 128), e.rand(20, 2, 128), e.rand(20, 2, 128)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda x: e.be.forward(x, k, v, e.mods[0], b), q, check_trace=False)
    assert not e.kvp.k_codes.any()  # nothing stored
    assert not e.be.forward(q, k, v, e.mods[0], b).isnan().any()


def test_phases_are_the_step_in_two(cuda):
    e = Engine(cuda, "quest", 1, 8, 2, 128, torch.bfloat16, 2, 900, 30)
    e.prefill([0, 1], [500, 70])
    rpi, seq = i64([0, 1], cuda), i64([501, 71], cuda)
    loc, pos = e.rtp.assign_decode(rpi, seq)
    batch = ForwardBatch(ForwardMode.DECODE, None, pos, rpi, seq, loc, e.rtp, e.kvp, e.be)
    e.be.init_forward_metadata(batch)
    q, k, v = e.rand(2, 8, 128), e.rand(2, 2, 128), e.rand(2, 2, 128)
    whole = e.be.forward(q, k, v, e.mods[0], batch)
    e.be.forward_decode_phase(q, k, v, e.mods[0], batch, 1)
    assert torch.equal(whole, e.be.forward_decode_phase(q, k, v, e.mods[0], batch, 2))
    with pytest.raises(ValueError, match="phase"):
        e.be.forward_decode_phase(q, k, v, e.mods[0], batch, 4)
    with pytest.raises(ValueError, match="block"):
        e.be.sparse_attention(q, e.mods[0], rpi, torch.zeros(2, 256, dtype=torch.int32, device=cuda), seq.int(), 2)


@pytest.mark.parametrize("lens, top_k, width, heads, avoid", [
    ([5000], 2048, 6000, 32, False), ([64 * 40 + 1, 64, 0, 700, 513, 512, 3000], 512, 4000, 8, True),
    ([1500 + 97 * i for i in range(30)], 512, 66000, 24, False), ([600 + i for i in range(64)], 512, 700, 16, False),
    ([1, 64, 130, 2000] * 16, 1024, 40000, 32, False), ([600] * 65, 512, 700, 16, False), ([9000, 4161, 4160], 4160, 9001, 32, True),
    ([2000] * 5, 448, 3000, 32, False), ([70000, 300], 2048, 530000, 32, False), ([900, 500, 60], 512, 512, 8, False)])
def test_a_divided_step_of_quest(cuda, lens, top_k, width, heads, avoid):
    """With the step's division, at the shape of two launches and beside it: selections, cache and
    answers, to the bit, of the three launches."""
    kv, dim, bs = 4, 128, len(lens)
    gen = torch.Generator(device=cuda).manual_seed(bs)
    rtp = BlockReqToTokenPool(bs + 1, width, sum(n // 64 + 2 for n in lens) + 5, cuda)
    kvp = Fp8TokenToKVPool(rtp.num_blocks, 1, kv, dim, cuda)
    be = QuestOnlyBackend(rtp, kvp, {"algorithm": "quest", "top_k": top_k, "quest_page_size": 64, "avoid_recent_overlap": avoid})
    be.quest.trace = QuestTrace()
    reqs, had = torch.arange(bs, device=cuda) + 1, [min(max(n - 1, 0), width) for n in lens]
    total = sum(had)
    loc, _ = rtp.assign(reqs, i64([0] * bs, cuda), i64(had, cuda), total)
    pages = torch.randn(total // 64 + 1, kv, dim, device=cuda, generator=gen).repeat_interleave(64, 0)[:total]
    kvp.set_kv_buffer(0, loc, pages + torch.randn(total, kv, dim, device=cuda, generator=gen),
                      torch.randn(total, kv, dim, device=cuda, generator=gen))
    be.quest.update_prefill_representations_blocks(reqs, i64(had, cuda), kvp, rtp.block_table)
    rtp.check_errors()
    seq = i64([min(n, width) for n in lens], cuda)
    for step in range(3):
        loc, pos = rtp.assign_decode(reqs, seq)
        batch = ForwardBatch(ForwardMode.DECODE, None, pos, reqs, seq, loc, rtp, kvp, be)
        q, k, v = (torch.randn(bs, h, dim, device=cuda, generator=gen).bfloat16() for h in (heads, kv, kv))
        if step == 2:
            q[:] = 0  # every page scores alike
        be.init_forward_metadata(batch)
        be._positions.fill_(-7)
        out = be.forward(q, k, v, Layer(0, dim), batch)
        got = be._positions.clone(), kvp.k_codes.clone(), kvp.v_codes.clone(), kvp.k_scale.clone(), kvp.v_scale.clone()
        be.quest._step.plan = None
        be._positions.fill_(-7)
        want = be.forward(q, k, v, Layer(0, dim), batch)
        assert torch.equal(out, want) and not out.isnan().any()
        for a, b in zip(got, (be._positions, kvp.k_codes, kvp.v_codes, kvp.k_scale, kvp.v_scale)):
            assert torch.equal(a, b)
        seq = torch.where((seq > 0) & (seq < width), seq + 1, seq)
    rtp.check_errors()


@pytest.mark.parametrize("lens, top_k, width, avoid", [
    ([200000, 700, 1, 164000], 2048, 200000, False),    # 3125 pages: more than 2560, which a block selects of in one form less
    ([3000, 66, 1500, 900], 1024, 200000, True),        # the same table with few candidates
    ([262208, 70000], 2624, 262208, True),              # 4097 pages: past what a begin launch selects of
    ([524288, 300], 2048, 524288, False),               # 8192 pages, the most that a block selects of
    ([524352, 5000], 512, 524352, False),               # one more
    ([40000, 3000, 64], 2624, 40001, False), ([40000, 3000, 64], 2688, 40001, True),  # 40 pages and one more
    ([270000, 5000], 4160, 270000, False), ([5000, 6000], 4160, 180000, False)])  # 64 pages
def test_selections_in_wide_tables(cuda, lens, top_k, width, avoid):
    """Selections of every form that a step over many pages takes: the oracle's positions, in two launches
    and in three, and the same answers; pages with scores of their own, and all alike."""
    kv, dim, heads, bs = 4, 128, 16, len(lens)
    gen = torch.Generator(device=cuda).manual_seed(width + top_k)
    rtp = BlockReqToTokenPool(bs, width, sum(n // 64 + 2 for n in lens) + 1, cuda)
    kvp = Fp8TokenToKVPool(rtp.num_blocks, 1, kv, dim, cuda)
    be = QuestOnlyBackend(rtp, kvp, {"algorithm": "quest", "top_k": top_k, "quest_page_size": 64, "avoid_recent_overlap": avoid})
    reqs, had = torch.arange(bs, device=cuda), [n - 1 for n in lens]
    for r, n in enumerate(had):  # (a request at a time: the values are made in float32)
        if n == 0:
            continue
        loc, _ = rtp.assign(i64([r], cuda), i64([0], cuda), i64([n], cuda), n)
        x = torch.randn(n // 64 + 1, kv, dim, device=cuda, generator=gen).repeat_interleave(64, 0)[:n].to(torch.bfloat16)
        kvp.set_kv_buffer(0, loc, x + torch.randn(n, kv, dim, device=cuda, generator=gen).to(torch.bfloat16),
                          torch.randn(n, kv, dim, device=cuda, generator=gen).to(torch.bfloat16))
    be.quest.update_prefill_representations_blocks(reqs, i64(had, cuda), kvp, rtp.block_table)
    rtp.check_errors()
    seq = i64(lens, cuda)
    loc, pos = rtp.assign_decode(reqs, seq)
    batch = ForwardBatch(ForwardMode.DECODE, None, pos, reqs, seq, loc, rtp, kvp, be)
    for alike in (False, True):
        q, k, v = (torch.randn(bs, h, dim, device=cuda, generator=gen).bfloat16() for h in (heads, kv, kv))
        if alike:
            q[:] = 0
        be.init_forward_metadata(batch)
        outs = []
        for planned in (True, False):
            if not planned:
                be.quest._step.plan = None
            be._positions.fill_(-7)
            outs.append((be.forward(q, k, v, Layer(0, dim), batch), be._positions.clone()))
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1]) and not outs[0][0].isnan().any()
        qbar = oq.group_queries(q.float().cpu().numpy(), kv, dim, True)
        for i, s in enumerate(lens):
            if s <= top_k:
                want = np.arange(s)
            else:
                full = (s - 1) // 64
                words = be.quest.page_k_bounds[0, i, :full].view(torch.int16).cpu().numpy().view(np.uint16)
                limit = s // 64 - 1 if avoid else s // 64
                pages = oq.topk_pages(oq.page_scores(qbar[i : i + 1], words[None])[0], min(limit, full), top_k // 64 - 1)
                want = np.concatenate([(pages[:, None] * 64 + np.arange(64)).reshape(-1), np.arange(s - 64, s)])
            assert outs[0][1][i, : len(want)].tolist() == want.tolist(), (i, alike)


def test_pools_that_do_not_go_together(cuda):
    paged, rows = BlockReqToTokenPool(2, 300, 9, cuda), ReqToTokenPool(2, 300, cuda)
    fp8, plain = Fp8TokenToKVPool(9, 1, 2, 128, cuda), MHATokenToKVPool(600, 1, 2, 128, torch.bfloat16, cuda)
    cfg = {"algorithm": "quest", "top_k": 128, "quest_page_size": 64}
    with pytest.raises(ValueError, match="BlockReqToTokenPool"):
        DenseBackend(rows, fp8)
    with pytest.raises(ValueError, match="blocks"):
        DenseBackend(BlockReqToTokenPool(2, 300, 10, cuda), fp8)
    with pytest.raises(ValueError, match="quest_page_size must be 64"):
        QuestOnlyBackend(paged, fp8, {**cfg, "quest_page_size": 32})
    with pytest.raises(ValueError, match="MHATokenToKVPool"):
        QuestHiSparseBackend(paged, fp8, cfg, host_pool_size=100)
    DenseBackend(paged, plain)


@pytest.mark.parametrize("backend", ["dense", "quest"])
def test_paged_rows_serve_the_bf16_pool(cuda, backend):
    """The slot maps with an MHATokenToKVPool: the same outputs as with rows handed out by hand."""
    outs = []
    for paged in (True, False):
        gen = torch.Generator(device=cuda).manual_seed(1)
        rtp = BlockReqToTokenPool(2, 600, 20, cuda) if paged else ReqToTokenPool(2, 600, cuda)
        kvp = MHATokenToKVPool(20 * 64, 1, 4, 128, torch.bfloat16, cuda)
        be = (DenseBackend(rtp, kvp) if backend == "dense" else
              QuestOnlyBackend(rtp, kvp, {"algorithm": "quest", "top_k": 128, "quest_page_size": 64}))
        rpi, pre, ext = i64([1, 0], cuda), i64([0, 0], cuda), i64([300, 90], cuda)
        if paged:
            loc, _ = rtp.assign(rpi, pre, ext, 390)
        else:
            loc = torch.arange(1, 391, device=cuda)
            rtp.req_to_token[1, :300], rtp.req_to_token[0, :90] = loc[:300].int(), loc[300:].int()
        batch = ForwardBatch(ForwardMode.EXTEND, None, None, rpi, ext, loc, rtp, kvp, be, extend_prefix_lens=pre, extend_seq_lens=ext)

        def rand(*shape):
            return torch.empty(shape, device=cuda).normal_(generator=gen).to(torch.bfloat16)

        got = [be.forward(rand(390, 16, 128), rand(390, 4, 128), rand(390, 4, 128), Layer(0, 128), batch)]
        seq = i64([301, 91], cuda)
        if paged:
            loc, _ = rtp.assign_decode(rpi, seq)
        else:
            loc = i64([500, 501], cuda)
            rtp.req_to_token[rpi, seq - 1] = loc.int()
        batch = ForwardBatch(ForwardMode.DECODE, None, None, rpi, seq, loc, rtp, kvp, be)
        be.init_forward_metadata(batch)
        got.append(be.forward(rand(2, 16, 128), rand(2, 4, 128), rand(2, 4, 128), Layer(0, 128), batch))
        outs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_blocks_past_32_bit_offsets(cuda):
    """A layer of more than 2^32 bytes of codes: its last blocks written, read, bounded and attended."""
    from qwenquest_amd.attention.ops import fp8_decode_attention, fp8_extend_attention

    kv, dim, blocks = 8, 128, 70_000  # 65536 bytes a block
    pool = Fp8TokenToKVPool(blocks, 1, kv, dim, cuda)
    assert pool.k_codes[0].numel() > 1 << 32
    ids = [blocks - 1, 1, blocks - 2, blocks // 2]
    table = torch.tensor([ids], dtype=torch.int32, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(0)
    loc = torch.tensor([b * 64 + t for b in ids for t in range(64)], device=cuda)
    k, v = (torch.empty((256, kv, dim), device=cuda).normal_(generator=gen).to(torch.bfloat16) for _ in range(2))
    pool.set_kv_buffer(0, loc, k, v)
    cache = of.Cache(5, kv, dim)  # the same in small blocks
    cache.write(torch.arange(64, 320).numpy(), k.float().cpu().numpy(), v.float().cpu().numpy())
    kw, vw = cache.rows(np.arange(64, 320))
    got = pool.get_rows(0, loc, torch.float32)
    assert np.array_equal(got[0].cpu().numpy(), kw) and np.array_equal(got[1].cpu().numpy(), vw)
    q = torch.empty((2, 16, dim), device=cuda).normal_(generator=gen).to(torch.bfloat16)
    scale, n = dim**-0.5, 230
    for out, row, seen in (
            (fp8_decode_attention(q[:1], pool, 0, table, i64([0], cuda), i64([n], cuda), scale), q[0], n),
            (fp8_extend_attention(q, pool, 0, table, i64([0], cuda), i64([n], cuda), i64([n - 2], cuda), i64([2], cuda), scale)[1:], q[1], n)):
        want, spread, size = of.attend(row.double().cpu().numpy(), kw[:seen], vw[:seen], scale)
        tol = of.attend_tolerance(want, spread, size, seen, dim, True, 12)
        assert (np.abs(out[0].double().cpu().numpy().reshape(want.shape) - want) <= tol).all()
    from qwenquest_amd.quest import QuestAlgorithm

    quest = QuestAlgorithm(128, 64, cuda)
    quest.init_storage(0, 1, 1, 256, kv, dim)
    quest.update_prefill_representations_blocks(i64([0], cuda), i64([256], cuda), pool, table)
    b = quest.page_k_bounds[0, 0].float().cpu().numpy()
    pages = kw.reshape(4, 64, kv, dim)
    assert np.array_equal(b[..., 0], pages.min(1)) and np.array_equal(b[..., 1], pages.max(1))
