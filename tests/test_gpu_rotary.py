"""Head norms with the position rotation, against float64.

Tolerance, of a head's outputs, in units of the larger of a pair (h = sqrt(a^2 + b^2) bounds both outputs): half a step
of the output's type, and in float32 the norm (a sum of D squares, partial sums half a step each, by lanes of 8 and
halving: under 16 steps, of which the root takes half; root, product and weight 4 half steps), the angle's sine and cosine
(2^-22 absolute: 2 steps of the function and the reduction) and three roundings of the rotation."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qwenquest_amd import QKNormRotary
from qwenquest_amd.attention import DenseBackend
from qwenquest_amd.batch import ForwardBatch, ForwardMode
from qwenquest_amd.memory import MHATokenToKVPool, ReqToTokenPool

pytestmark = pytest.mark.gpu


def deal(sections, cycled):
    left = list(sections)
    if not cycled:
        return [a for a, m in enumerate(left) for _ in range(m)]
    out = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def want(x, w, eps, freq, axis, pos, neighbours):
    """x [n, heads, D] in float64, and each output's size."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w
    P = len(freq)
    at = np.arange(P)
    a, b = (2 * at, 2 * at + 1) if neighbours else (at, at + P)
    t = pos[axis, :].T[:, None].astype(np.float64) * freq
    out, size = y.copy(), np.abs(y)
    if P:
        out[..., a] = y[..., a] * np.cos(t) - y[..., b] * np.sin(t)
        out[..., b] = y[..., b] * np.cos(t) + y[..., a] * np.sin(t)
        size[..., a] = size[..., b] = np.hypot(y[..., a], y[..., b])
    return out, size


def check(got, x, w, eps, freq, axis, pos, neighbours, far=1.0):
    ref, size = want(x.double().cpu().numpy(), None if w is None else w.double().cpu().numpy(), eps, np.asarray(freq),
                     np.asarray(axis, dtype=np.int64), pos, neighbours)
    half = 2.0**-8 if x.dtype == torch.bfloat16 else 2.0**-24
    # far: what float64 itself leaves of an angle of that many turns
    tol = half * np.abs(ref) + (16 * 2.0**-24 + 2.0**-22 + far * 2.0**-51) * size + 1e-37
    err = np.abs(got.double().cpu().numpy() - ref)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert (err <= tol).all(), f"off by {(err / tol).max():.2f} tolerances"


CASES = [  # heads, kv, dim, rotary_dim, sections, cycled, pairs
    (32, 4, 128, 128, None, False, "halves"), (32, 4, 128, 128, (24, 20, 20), True, "halves"), (14, 2, 64, 32, (4, 6, 6), False, "neighbours"),
    (1, 1, 8, 8, None, False, "neighbours"), (3, 3, 16, 16, None, False, "halves"), (5, 1, 80, 80, (20, 20), True, "halves"),
    (7, 7, 96, 48, None, False, "halves"), (8, 2, 256, 256, (128, 0, 0), False, "halves"), (2, 1, 512, 64, None, False, "neighbours"),
    (6, 2, 512, 512, None, False, "halves"), (16, 8, 40, 0, None, False, "halves"), (9, 3, 24, 16, None, False, "halves")]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("n", [1, 3, 129, 5000])
def test_shapes(cuda, n, case, dtype):
    heads, kv, dim, rot, sections, cycled, pairs = case
    gen = torch.Generator(device=cuda).manual_seed(dim + n)
    wq, wk = (1 + torch.empty(dim, device=cuda).normal_(generator=gen) * 0.3 for _ in range(2))
    op = QKNormRotary(heads, kv, dim, q_weight=wq, k_weight=wk, eps=1e-6, base=1e6, rotary_dim=rot, sections=sections,
                      section_order="cycled" if cycled else "blocks", pairs=pairs, device=cuda)
    qkv = torch.empty((n, (heads + 2 * kv) * dim), device=cuda).normal_(generator=gen)
    qkv = (qkv * torch.exp(torch.empty((n, 1), device=cuda).normal_(generator=gen))).to(dtype)
    axes = len(sections) if sections else 1
    pos = torch.randint(0, 40000, (axes, n), device=cuda, generator=gen)
    q, k, v = op(qkv, pos if axes > 1 else pos[0])
    x = qkv.view(n, -1, dim)
    freq = 1e6 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    axis = deal(sections or (rot // 2,), cycled)
    p = pos.cpu().numpy()
    few = slice(None) if n < 1000 else slice(0, n, 37)
    for got, part, w in ((q, x[:, :heads], wq), (k, x[:, heads : heads + kv], wk)):
        check(got[few].contiguous(), part[few], w, 1e-6, freq, axis, p[:, few], pairs == "neighbours")
    assert torch.equal(v, x[:, heads + kv :]) and v.is_contiguous()


@pytest.mark.parametrize("norm", [(True, False), (False, True), (False, False)])
def test_norms_left_out(cuda, norm):
    w = torch.rand(64, device=cuda) + 0.5
    op = QKNormRotary(4, 2, 64, q_weight=w if norm[0] else None, k_weight=w if norm[1] else None, eps=1e-3, device=cuda)
    qkv, pos = torch.randn(50, 8 * 64, device=cuda), torch.arange(50, device=cuda)
    q, k, _ = op(qkv, pos)
    freq, p = 10000.0 ** (-np.arange(32) / 32.0), pos.cpu().numpy()[None]
    x = qkv.view(50, 8, 64)
    check(q, x[:, :4], w if norm[0] else None, 1e-3, freq, [0] * 32, p, False)
    check(k, x[:, 4:6], w if norm[1] else None, 1e-3, freq, [0] * 32, p, False)


def test_far_positions(cuda):
    """Angles of up to 2^31 radians, and past them NaN where a channel turns; negative positions."""
    pos = np.array([0, 1, -1, 131071, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31) + 1, 1 << 31, -(1 << 31), 1 << 62, -(1 << 62)])
    op = QKNormRotary(2, 1, 64, rotary_dim=32, base=1e4, device=cuda)
    qkv = torch.randn(len(pos), 4 * 64, device=cuda)
    q, k, v = op(qkv, torch.from_numpy(pos).to(cuda))
    freq = 1e4 ** (-2.0 * np.arange(16) / 32)
    x = qkv.view(-1, 4, 64)
    # the reference's own angle, and the kernel's, are off by half a step of float64: 2^-53 of 2^31
    check(q[:8].contiguous(), x[:8, :2], None, 0.0, freq, [0] * 16, pos[None, :8], False, far=2.0**31)
    assert q[8:, :, :32].isnan().all() and k[8:, :, :32].isnan().all()
    assert torch.equal(q[8:, :, 32:], x[8:, :2, 32:]) and torch.equal(v, x[:, 3:])
    near = 6
    check(q[:near].contiguous(), x[:near, :2], None, 0.0, freq, [0] * 16, pos[None, :near], False, far=2.0**25)


def test_given_frequencies_and_every_angle(cuda):
    """Angles all round the circle, close to its quarters too, by frequencies of any size and sign."""
    freq = np.concatenate([np.pi / 2 * np.array([1, -1, 2, 3, 4, 0.5, 1.5, 0]), np.array([100.0, -7.3, 1e-9, 1e-300, 0.1, 1.0, 2.0, 1e5])])
    op = QKNormRotary(1, 1, 32, inv_freq=torch.from_numpy(freq), device=cuda)
    qkv, pos = torch.randn(300, 3 * 32, device=cuda), np.arange(-150, 150)
    q, _, _ = op(qkv, torch.from_numpy(pos).to(cuda))
    check(q, qkv.view(300, 3, 32)[:, :1], None, 0.0, freq, [0] * 16, pos[None], False, far=2.0**24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_of_any_size(cuda, dtype):
    """Zeros, tiny and large rows, infinities and NaN, each in a head of its own."""
    op = QKNormRotary(6, 1, 64, q_weight=torch.ones(64), k_weight=torch.ones(64), eps=1e-6, device=cuda)
    x = torch.randn(1, 8, 64, device=cuda)
    for h, s in enumerate((0.0, 1e-20, 1e15, 1.0, 1.0, 3.0)):
        x[0, h] *= s
    x[0, 3, 7], x[0, 4, 9] = float("inf"), float("nan")
    x = x.to(dtype)
    q, k, v = op(x.view(1, -1), torch.tensor([5], device=cuda))
    freq, p = 1e4 ** (-np.arange(32) / 32.0), np.array([[5]])
    ok = [0, 1, 2, 5]
    check(q[:, ok].contiguous(), x[:, ok], torch.ones(64), 1e-6, freq, [0] * 32, p, False)
    assert not q[0, 0].any() and q[0, 3].isnan().any() and q[0, 4].isnan().all()
    assert not k.isnan().any() and torch.equal(v, x[:, 7:])


def test_strides_alignments_and_types_of_its_inputs(cuda):
    w = torch.rand(64, device=cuda, dtype=torch.bfloat16) + 0.5
    op = QKNormRotary(4, 2, 64, q_weight=w, k_weight=w, device=cuda)
    dense, pos = torch.randn(33, 8 * 64, device=cuda).to(torch.bfloat16), torch.arange(33, device=cuda)
    ref = op(dense, pos)
    wide = torch.zeros(33, 8 * 64 + 8, device=cuda, dtype=torch.bfloat16)
    wide[:, :-8] = dense
    odd = torch.zeros(33, 8 * 64 + 3, device=cuda, dtype=torch.bfloat16)
    odd[:, 3:] = dense
    last = torch.zeros(33, 8 * 64, 2, device=cuda, dtype=torch.bfloat16)
    last[..., 1] = dense
    rows = torch.zeros(66, 8 * 64, device=cuda, dtype=torch.bfloat16)
    rows[::2] = dense
    for x, p in ((wide[:, :-8], pos), (odd[:, 3:], pos.int()), (last[..., 1], pos.cpu()), (rows[::2], pos[None]),
                 (dense.flip(0).flip(0), pos.short())):
        assert all(torch.equal(a, b) for a, b in zip(op(x, p), ref))
    x3 = dense.view(33, 8, 64)
    one = dense[:1, :].expand(33, -1)  # a broadcast row
    same = op(one, pos)
    assert torch.equal(same[0][:1], ref[0][:1]) and torch.equal(same[1], op(one.contiguous(), pos)[1])
    for q, k in ((x3[:, :4], x3[:, 4:6]), (dense[:, :256], x3[:, 4:6].clone()), (x3[:, :4].transpose(0, 1).contiguous().transpose(0, 1), x3[:, 4:6])):
        got = op.apply(q, k, pos)
        assert len(got) == 2 and torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    empty = op(dense[:0], pos[:0])
    assert [tuple(t.shape) for t in empty] == [(0, 4, 64), (0, 2, 64), (0, 2, 64)]
    copied = torch.ones(64, device=cuda)
    held = QKNormRotary(4, 2, 64, q_weight=copied, device=cuda)
    a = held(dense, pos)[0]
    copied.zero_()
    assert torch.equal(held(dense, pos)[0], a)


def test_what_is_refused(cuda):
    def make(**kw):
        return QKNormRotary(**{**dict(num_heads=4, kv_heads=2, head_dim=64, device=cuda), **kw})

    for kw, said in ((dict(num_heads=0), "heads"), (dict(head_dim=60), "multiple of 8"), (dict(head_dim=520), "multiple of 8"),
                     (dict(pairs="quarters"), "pairs"), (dict(section_order="x"), "section_order"), (dict(rotary_dim=72), "rotary_dim"),
                     (dict(rotary_dim=24), "multiple of 16"), (dict(rotary_dim=20, pairs="neighbours"), "multiple of 8"),
                     (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(base=0.0), "base"), (dict(inv_freq=[1.0]), "inv_freq"),
                     (dict(inv_freq=[float("inf")] * 32), "inv_freq"), (dict(sections=(10, 10)), "sections"), (dict(sections=(-1, 33)), "sections"),
                     (dict(sections=()), "sections"), (dict(q_weight=torch.ones(32)), "q_weight"), (dict(k_weight=torch.ones(64).int()), "k_weight")):
        with pytest.raises(ValueError, match=said):
            make(**kw)
    with pytest.raises(RuntimeError, match="GPU"):
        make(device="cpu")
    op = make(sections=(16, 8, 8))
    x, pos = torch.zeros(5, 512, device=cuda), torch.zeros(3, 5, dtype=torch.int64, device=cuda)
    for a, said in (((x[:, :500], pos), "qkv"), ((x.view(5, 8, 64), pos), "qkv"), ((x, pos[0]), "positions"), ((x, pos[:, :4]), "positions"),
                    ((x, pos.float()), "whole"), ((x.half(), pos), "dtype"), ((x.cpu(), pos), "lie on")):
        with pytest.raises(ValueError, match=said):
            op(*a)
    y = x.view(5, 8, 64)
    for a, said in (((y[:, :3], y[:, 4:6], pos), "q must"), ((y[:, :4], y[:4, 4:6], pos), "differ"), ((y[:, :4], y[:, 4:6].bfloat16(), pos), "differ")):
        with pytest.raises(ValueError, match=said):
            op.apply(*a)
    with pytest.raises(RuntimeError, match="no gradients"):
        op(x.clone().requires_grad_(), pos)
    with torch.no_grad():
        op(x.clone().requires_grad_(), pos)


def test_a_tangent_is_refused(cuda):
    op = QKNormRotary(2, 1, 64, device=cuda)
    x, pos = torch.zeros(3, 256, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no gradients"):
            op(dual, pos)
        with pytest.raises(RuntimeError, match="no gradients"):
            op.apply(dual[:, :128], x[:, 128:192], pos)
        op(x, pos)


def test_captured_and_on_another_stream(cuda):
    w = torch.rand(128, device=cuda) + 0.5
    op = QKNormRotary(8, 2, 128, q_weight=w, k_weight=w, base=1e6, device=cuda)
    qkv, pos = torch.zeros(40, 12 * 128, device=cuda, dtype=torch.bfloat16), torch.zeros(40, dtype=torch.int64, device=cuda)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        op(qkv, pos)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op(qkv, pos)
    for i in range(3):
        qkv.normal_()
        pos.random_(0, 1 << 20)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, op(qkv, pos)))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            other = op(qkv, pos)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, other))


def test_rotation_makes_scores_depend_on_distance(cuda):
    """q k of rotated heads depends on the two positions' difference alone."""
    op = QKNormRotary(1, 1, 128, base=1e6, device=cuda)
    q, k = (torch.randn(1, 1, 128, device=cuda).expand(8, 1, 128) for _ in range(2))
    at = torch.tensor([0, 1, 100, 5000, 131072, 1 << 20, 1 << 24, (1 << 31) - 50], device=cuda)
    a, _ = op.apply(q, k, at + 37)
    _, b = op.apply(q, k, at)
    s = (a.double() * b.double()).sum(-1)[:, 0]
    size = (a.double().abs() * b.double().abs()).sum(-1)[:, 0]
    assert ((s - s[0]).abs() <= 2 * (3 * 2.0**-24 + 2.0**-22) * (size + size[0]) * 2**0.5).all()


def test_forward_qkv_is_the_norms_then_forward(cuda):
    """A layer's attention from its QKV product, in prefill and in decode steps."""

    class Layer:
        layer_id, scaling = 0, 64**-0.5
        rotary = QKNormRotary(8, 2, 64, q_weight=torch.rand(64) + 0.5, k_weight=torch.rand(64) + 0.5, device=cuda)

    outs = []
    for fused in (True, False):
        rtp, kvp = ReqToTokenPool(2, 64, cuda), MHATokenToKVPool(128, 1, 2, 64, torch.bfloat16, cuda)
        rtp.req_to_token[:] = torch.arange(1, 129, device=cuda, dtype=torch.int32).view(2, 64)
        be = DenseBackend(rtp, kvp)
        gen = torch.Generator(device=cuda).manual_seed(1)
        rpi = torch.arange(2, device=cuda)
        for step in range(3):
            n = 40 if step == 0 else 2
            qkv = torch.empty((n, 12 * 64), device=cuda).normal_(generator=gen).to(torch.bfloat16)
            if step == 0:
                seq, pos = torch.tensor([25, 15], device=cuda), torch.cat([torch.arange(25), torch.arange(15)]).to(cuda)
                loc = torch.cat([rtp.req_to_token[0, :25], rtp.req_to_token[1, :15]]).long()
                batch = ForwardBatch(ForwardMode.EXTEND, None, pos, rpi, seq, loc, rtp, kvp, be,
                                     extend_prefix_lens=torch.zeros_like(seq), extend_seq_lens=seq)
            else:
                seq = torch.tensor([25 + step, 15 + step], device=cuda)
                loc = rtp.req_to_token[rpi, seq - 1].long()
                batch = ForwardBatch(ForwardMode.DECODE, None, seq - 1, rpi, seq, loc, rtp, kvp, be)
            be.init_forward_metadata(batch)
            if fused:
                outs.append(be.forward_qkv(qkv, Layer, batch))
            else:
                assert torch.equal(be.forward(*Layer.rotary(qkv, batch.positions), Layer, batch), outs[step])
    assert all(o.isfinite().all() for o in outs)

    class Bare:
        layer_id, scaling = 0, 0.1

    with pytest.raises(ValueError, match="rotary"):
        be.forward_qkv(qkv, Bare, batch)
    batch.positions = None
    with pytest.raises(ValueError, match="positions"):
        be.forward_qkv(qkv, Layer, batch)
