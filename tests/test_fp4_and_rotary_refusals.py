"""Refusals of the 4-bit cache's and the rotation's entry points.  No GPU: every call here is refused before a
kernel is launched.  And the 4-bit cache's oracle."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import fp4_cache as o4
from qwenquest_amd import _lib
from qwenquest_amd.paged import CodedTokenToKVPool, Fp4TokenToKVPool
from qwenquest_amd.rotary import QKNormRotary
from tests.test_block_pools import BAD_CACHE, CACHE, FAKE, lib, refused  # noqa: F401 - lib: a fixture

ODD = ctypes.c_void_p(4104)


def test_both_need_a_gpu():
    with pytest.raises(RuntimeError, match="Fp4TokenToKVPool needs a GPU"):
        Fp4TokenToKVPool(5, 1, 4, 128, "cpu")
    with pytest.raises(RuntimeError, match="QKNormRotary needs a GPU"):
        QKNormRotary(4, 1, 128, device="cpu")
    assert issubclass(Fp4TokenToKVPool, CodedTokenToKVPool)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [
    (dict(dtype=2), b"dtype"), (dict(n=-1), b"bad sizes"), (dict(n=1 << 31), b"bad sizes"), (dict(k=None), b"null"), (dict(loc=None), b"null"),
    (dict(k=ODD), b"aligned"), (dict(v=ODD), b"aligned"), (dict(n=(1 << 31) - 1, kv=1024), b"bad sizes")])
def test_store_refuses(lib, kw, said):  # noqa: F811
    a = {**CACHE, **dict(k=FAKE, v=FAKE, dtype=0, loc=FAKE, n=3), **kw}
    refused(lib.qq_fp4_store(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [(dict(dtype=2), b"dtype"), (dict(n=-1), b"bad sizes"), (dict(k=None), b"null"),
                                                  (dict(loc=None), b"null"), (dict(n=(1 << 31) - 1, kv=1024), b"bad sizes")])
def test_rows_refuses(lib, kw, said):  # noqa: F811
    a = {**CACHE, **dict(loc=FAKE, n=3, k=FAKE, v=FAKE, dtype=0), **kw}
    refused(lib.qq_fp4_rows(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", [
    (dict(kc=None), b"null cache"), (dict(ks=None), b"null cache"), (dict(dim=80), b"head_dim"), (dict(bs=-1), b"bad sizes"),
    (dict(bs=65536), b"bad sizes"), (dict(layers=0), b"bad sizes"), (dict(reqs=0), b"bad sizes"), (dict(mp=0), b"bad sizes"),
    (dict(tstride=3), b"bad sizes"), (dict(seq=None), b"null"), (dict(bounds=None), b"null"), (dict(table=None), b"null"),
    (dict(actual=FAKE), b"layout"), (dict(plan=FAKE, plan_bytes=1 << 30), b"decode step"),
    (dict(plan=FAKE, plan_bytes=1 << 30, decode=1, top_k=100), b"decode step"), (dict(plan=FAKE, plan_bytes=9, decode=1), b"workspace"),
    (dict(plan=FAKE, plan_bytes=1 << 30, decode=1, bs=65535, tcols=1 << 24, tstride=1 << 24), b"units")])
def test_page_bounds_refuses(lib, kw, said):  # noqa: F811
    a = dict(kc=FAKE, kst=100, ks=FAKE, sst=10, blocks=5, kv=4, dim=128, table=FAKE, tstride=4, trows=2, tcols=4, rpi=FAKE,
             seq=FAKE, prefix=None, bs=2, decode=0, max_new=0, layers=1, bounds=FAKE, reqs=2, mp=4, top_k=128,
             avoid=0, actual=None, limit=None, plan=None, plan_bytes=0)
    a.update(kw)
    refused(lib.qq_fp4_page_bounds(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [
    (dict(qd=2), b"dtype"), (dict(H=30), b"divisible"), (dict(H=0), b"divisible"), (dict(bs=-1), b"bad sizes"),
    (dict(tstride=3), b"bad sizes"), (dict(trows=0), b"bad sizes"), (dict(pos=FAKE, top_k=100), b"multiple"),
    (dict(pos=FAKE, top_k=128, pstride=64), b"multiple"), (dict(q=None), b"null"), (dict(out=None), b"null"),
    (dict(q=ODD), b"aligned"), (dict(qst=4100), b"aligned"), (dict(bytes=64), b"workspace"), (dict(kn=FAKE), b"null"),
    (dict(bs=1 << 20, tcols=1 << 24, tstride=1 << 24), b"units"), (dict(planned=1, pos=FAKE, top_k=128, pstride=128), b"whole")])
def test_decode_refuses(lib, kw, said):  # noqa: F811
    a = dict(q=FAKE, qd=0, qst=4096, H=32, kn=None, vn=None, nd=0, loc=None, **CACHE, table=FAKE, tstride=4, trows=2, tcols=4,
             rpi=FAKE, seq=FAKE, bs=2, pos=None, pstride=0, top_k=0, scale=0.1, out=FAKE, ws=FAKE, bytes=1 << 30,
             planned=0)
    a.update(kw)
    refused(lib.qq_fp4_decode_attention(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", [
    (dict(blocks=0), b"blocks"), (dict(kv=0), b"KV heads"), (dict(dim=80), b"head_dim"), (dict(trows=0), b"bad sizes"),
    (dict(tcols=0), b"bad sizes"), (dict(bs=-1), b"bad sizes"), (dict(rpi=None), b"null"), (dict(seq=None), b"null"),
    (dict(ws=None), b"null"), (dict(bytes=64), b"workspace"), (dict(bs=1 << 20, tcols=1 << 24), b"units")])
def test_decode_plan_refuses(lib, kw, said):  # noqa: F811
    a = dict(blocks=5, kv=4, dim=128, trows=2, tcols=4, rpi=FAKE, seq=FAKE, bs=2, ws=FAKE, bytes=1 << 30)
    a.update(kw)
    refused(lib.qq_fp4_decode_plan(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [
    (dict(phase=0), b"phase"), (dict(phase=4), b"phase"), (dict(bounds=None), b"null"), (dict(scores=None), b"null"),
    (dict(pos=None), b"null"), (dict(limit=None), b"null"), (dict(layer=-1), b"bad sizes"), (dict(reqs=0), b"bad sizes"),
    (dict(top_k=100), b"multiple"), (dict(top_k=64 * 1026), b"selected pages"), (dict(kv=16, H=32), b"exceeds"),
    (dict(loc=None), b"null"), (dict(nd=7), b"dtype"), (dict(kn=ODD), b"aligned"), (dict(bytes=64), b"workspace")])
def test_quest_step_refuses(lib, kw, said):  # noqa: F811
    a = dict(q=FAKE, qd=0, qst=4096, H=32, kn=FAKE, vn=FAKE, nd=0, loc=FAKE, **CACHE, table=FAKE, tstride=4, trows=2, tcols=4,
             bounds=FAKE, layer=0, rpi=FAKE, seq=FAKE, limit=FAKE, bs=2, reqs=2, mp=4, top_k=128, scale=0.1, scores=FAKE, pos=FAKE,
             out=FAKE, ws=FAKE, bytes=1 << 30, phase=3, planned=0)
    a.update(kw)
    refused(lib.qq_fp4_quest_step(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [
    (dict(H=30), b"divisible"), (dict(scale=0.0), b"positive"), (dict(scale=float("nan")), b"positive"),
    (dict(scale=float("inf")), b"positive"), (dict(bs=-1), b"bad sizes"), (dict(n=1 << 28), b"bad sizes"),
    (dict(tstride=3), b"bad sizes"), (dict(q=None), b"null"), (dict(ext=None), b"null"), (dict(out=ODD), b"aligned"),
    (dict(n=8, tcols=1 << 12, tstride=1 << 12, ws=None), b"workspace")])
def test_extend_refuses(lib, kw, said):  # noqa: F811
    a = dict(q=FAKE, H=32, **CACHE, table=FAKE, tstride=4, trows=2, tcols=4, rpi=FAKE, seq=FAKE, prefix=FAKE, ext=FAKE, bs=2, n=10,
             scale=0.1, out=FAKE, ws=FAKE, bytes=1 << 30)
    a.update(kw)
    refused(lib.qq_fp4_extend_attention(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", [
    (dict(dtype=2), b"dtype"), (dict(dim=60), b"multiple of 8"), (dict(dim=520), b"multiple of 8"), (dict(dim=0), b"multiple of 8"),
    (dict(H=0), b"heads"), (dict(KV=0), b"heads"), (dict(H=65536), b"heads"), (dict(pairs=72), b"pairs"), (dict(pairs=12), b"multiples of 8"),
    (dict(pairs=10, neighbours=1), b"multiples of 4"), (dict(pairs=-8), b"pairs"), (dict(n=-1), b"bad sizes"), (dict(n=1 << 28), b"bad sizes"),
    (dict(axes=0), b"bad sizes"), (dict(q=None), b"null"), (dict(ko=None), b"null"), (dict(vo=None), b"null"), (dict(turns=None), b"null"),
    (dict(axis=None), b"null"), (dict(pos=None), b"null"), (dict(axes=2, ps=9), b"overlap"), (dict(q=ODD), b"aligned"), (dict(vo=ODD), b"aligned"),
    (dict(qs=4100), b"aligned"), (dict(ks=516), b"aligned"), (dict(dtype=1, vs=514), b"aligned")])
def test_rotary_refuses(lib, kw, said):  # noqa: F811
    a = dict(q=FAKE, qs=4096, k=FAKE, ks=512, v=FAKE, vs=512, dtype=0, H=32, KV=4, dim=128, n=10, wq=FAKE, wk=FAKE, eps=1e-6, turns=FAKE,
             axis=FAKE, pairs=64, neighbours=0, pos=FAKE, ps=10, axes=1, qo=FAKE, ko=FAKE, vo=FAKE)
    a.update(kw)
    refused(lib.qq_qk_norm_rotary(*a.values(), None), lib, said)


def test_no_launch_past_2_32_threads(lib):  # noqa: F811
    n = (1 << 30) - 63  # 2^24 blocks of 256
    refused(lib.qq_fp4_store(*{**CACHE, **dict(k=FAKE, v=FAKE, dtype=0, loc=FAKE, n=n)}.values(), None), lib, b"bad sizes")
    refused(lib.qq_fp4_rows(*{**CACHE, **dict(loc=FAKE, n=n, k=FAKE, v=FAKE, dtype=0)}.values(), None), lib, b"bad sizes")
    a = dict(q=FAKE, qs=8, k=FAKE, ks=8, v=None, vs=0, dtype=0, H=1, KV=1, dim=8, n=(1 << 26) - 4, wq=None, wk=None, eps=1e-6, turns=None,
             axis=None, pairs=0, neighbours=0, pos=None, ps=0, axes=1, qo=FAKE, ko=FAKE, vo=None)
    refused(lib.qq_qk_norm_rotary(*a.values(), None), lib, b"bad sizes")


def test_nothing_to_do(lib):  # noqa: F811
    assert lib.qq_fp4_store(*{**CACHE, **dict(k=None, v=None, dtype=0, loc=None, n=0)}.values(), None) == _lib.QQ_OK
    assert lib.qq_fp4_decode_workspace_bytes(0, 32, 4, 128) == 0 == lib.qq_fp4_decode_workspace_bytes(2, 30, 4, 128)
    small, large = (lib.qq_fp4_decode_workspace_bytes(bs, 32, 4, 128) for bs in (1, 1000))
    assert 0 < small < large < 32 << 20
    assert lib.qq_fp4_extend_workspace_bytes(0, 2, 32, 4, 128, 10) == 0


# ---------------------------------------------------------------- the oracle itself


def test_oracle_rounds_to_the_nearest_code():
    y = np.concatenate([np.linspace(-8, 8, 100001), (o4.GRID[1:] + o4.GRID[:-1]) / 2])
    got = o4.round_e2m1(y)
    grid = np.concatenate([-o4.GRID, o4.GRID])
    best = np.abs(y[:, None] - grid).min(1)
    assert np.allclose(np.abs(got - y), best, atol=0)
    assert np.isin(np.abs(got), o4.GRID).all()
    borders = o4.round_e2m1((o4.GRID[1:] + o4.GRID[:-1]) / 2)
    assert borders.tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]  # ties to the even code


def test_oracle_scales():
    assert o4.exponent(np.array([0.0, 7.0, np.nextafter(7.0, 8), 3.5, 1e-40, 3e38]), o4.K_EXP).tolist() == [-96, 0, 1, -1, -96, 125]
    assert o4.exponent(np.array([0.0, 7 * 2.0**59]), o4.V_EXP).tolist() == [-50, 59]
    c = o4.Cache(3, 1, 64)
    k, v = np.ones((2, 1, 64)), np.full((2, 1, 64), 0.7)
    k[0, 0, :32] = 100.0
    v[1, 0, 5] = np.inf
    c.write([64, 65], k, v)
    kw, vw = c.rows([64, 65])
    assert (kw[0, 0, :32] == 96.0).all() and (kw[0, 0, 32:] == 1.0).all() and (vw[0] == 0.75).all()
    assert np.isnan(kw[1]).all() and np.isnan(vw[1]).all()
    x = torch.randn(50, 2, 64, dtype=torch.float64).numpy()
    once = o4.quantise(x, 32, o4.K_EXP)
    top = np.abs(x.reshape(50, 2, 2, 32)).max(-1)
    # 2^e, half of the widest step (4 to 6, and 7 comes down to 6), is less than top / 3.5: e is the least with top <= 7 * 2^e
    assert (np.abs(once - x).reshape(50, 2, 2, 32).max(-1) <= top / 3.5).all()
