"""Refusals of the paged pools and the 8-bit cache's entry points, and their divisions of work.
No GPU: every call here is refused before a kernel is launched, or runs the host's rules."""

from __future__ import annotations

import ctypes
import os
import random
import subprocess

import numpy as np
import pytest
import torch

from oracle import fp8_cache as of
from qwenquest_amd import _lib
from qwenquest_amd.batch import DecodePlan
from qwenquest_amd.paged import BlockReqToTokenPool, Fp8TokenToKVPool
from tests.test_launch_shapes import CSRC, shutil

FAKE = ctypes.c_void_p(4096)  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from qwenquest_amd import build

        build.build()
    return _lib.load()


def test_pools_need_a_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        BlockReqToTokenPool(2, 128, 5, "cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        Fp8TokenToKVPool(5, 1, 4, 128, "cpu")


def assign(lib, **kw):
    a = dict(rpi=FAKE, lens=FAKE, new=FAKE, bs=2, total=10, table=FAKE, tstride=4, r2t=FAKE, rstride=256, width=256, reqs=4,
             held=FAKE, stack=FAKE, count=FAKE, cap=9, loc=FAKE, pos=FAKE, err=FAKE, mirror=None, ws=FAKE, bytes=1 << 20)
    a.update(kw)
    return lib.qq_block_assign(*a.values(), None)


@pytest.mark.parametrize("kw, said", [
    (dict(bs=-1), b"bad sizes"), (dict(total=-1), b"bad sizes"), (dict(total=1 << 31), b"bad sizes"),
    (dict(reqs=0), b"requests"), (dict(reqs=(1 << 18) + 1), b"requests"), (dict(width=0), b"table sizes"),
    (dict(rstride=255), b"table sizes"), (dict(tstride=3), b"table sizes"), (dict(cap=1 << 24), b"blocks"),
    (dict(rpi=None), b"null"), (dict(lens=None), b"null"), (dict(loc=None), b"null"), (dict(held=None), b"null"),
    (dict(new=None), b"one row per request"), (dict(bytes=8), b"workspace"), (dict(ws=None), b"workspace"),
    (dict(bs=0), b"no request"),
])
def test_assign_refuses(lib, kw, said):
    assert assign(lib, **kw) == _lib.QQ_EINVAL and said in lib.qq_last_error()


def test_assign_and_release_of_nothing(lib):
    assert assign(lib, bs=0, total=0) == _lib.QQ_OK
    args = [FAKE, 0, FAKE, 4, FAKE, 256, 256, 4, FAKE, FAKE, FAKE, 9, FAKE, None, FAKE, 1 << 20, None]
    assert lib.qq_block_release(*args) == _lib.QQ_OK
    args[1] = 3
    args[-2] = 16
    assert lib.qq_block_release(*args) == _lib.QQ_EINVAL and b"workspace" in lib.qq_last_error()


CACHE = dict(kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, blocks=5, kv=4, dim=128)
BAD_CACHE = [(dict(kc=None), b"null cache"), (dict(vs=None), b"null cache"), (dict(blocks=0), b"blocks"),
             (dict(blocks=(1 << 24) + 1), b"blocks"), (dict(kv=0), b"KV heads"), (dict(dim=96), b"head_dim"),
             (dict(dim=256), b"head_dim")]


def refused(status, lib, said):
    assert status == _lib.QQ_EINVAL and said in lib.qq_last_error(), lib.qq_last_error()


@pytest.mark.parametrize("kw, said", BAD_CACHE + [
    (dict(dtype=2), b"dtype"), (dict(n=-1), b"bad sizes"), (dict(k=None), b"null"), (dict(loc=None), b"null"),
    (dict(k=ctypes.c_void_p(4104)), b"aligned")])
def test_store_refuses(lib, kw, said):
    a = {**CACHE, **dict(k=FAKE, v=FAKE, dtype=0, loc=FAKE, n=3), **kw}
    refused(lib.qq_fp8_store(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [(dict(dtype=2), b"dtype"), (dict(n=-1), b"bad sizes"), (dict(k=None), b"null")])
def test_rows_refuses(lib, kw, said):
    a = {**CACHE, **dict(loc=FAKE, n=3, k=FAKE, v=FAKE, dtype=0), **kw}
    refused(lib.qq_fp8_rows(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", [
    (dict(kc=None), b"null cache"), (dict(dim=80), b"head_dim"), (dict(bs=-1), b"bad sizes"), (dict(bs=65536), b"bad sizes"),
    (dict(layers=0), b"bad sizes"), (dict(reqs=0), b"bad sizes"), (dict(mp=0), b"bad sizes"), (dict(tstride=3), b"bad sizes"),
    (dict(seq=None), b"null"), (dict(bounds=None), b"null"), (dict(table=None), b"null"), (dict(actual=FAKE), b"layout"), (dict(plan=FAKE, plan_bytes=1 << 30), b"decode step"),
    (dict(plan=FAKE, plan_bytes=1 << 30, decode=1, top_k=100), b"decode step"), (dict(plan=FAKE, plan_bytes=9, decode=1), b"workspace"),
    (dict(plan=FAKE, plan_bytes=1 << 30, decode=1, bs=65535, tcols=1 << 24, tstride=1 << 24), b"units")])
def test_page_bounds_refuses(lib, kw, said):
    a = dict(kc=FAKE, kst=100, ks=FAKE, sst=10, blocks=5, kv=4, dim=128, table=FAKE, tstride=4, trows=2, tcols=4, rpi=FAKE,
             seq=FAKE, prefix=None, bs=2, decode=0, max_new=0, layers=1, bounds=FAKE, reqs=2, mp=4, top_k=128,
             avoid=0, actual=None, limit=None, plan=None, plan_bytes=0)
    a.update(kw)
    refused(lib.qq_fp8_page_bounds(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [
    (dict(qd=2), b"dtype"), (dict(H=30), b"divisible"), (dict(H=0), b"divisible"), (dict(bs=-1), b"bad sizes"),
    (dict(tstride=3), b"bad sizes"), (dict(trows=0), b"bad sizes"), (dict(pos=FAKE, top_k=100), b"multiple"),
    (dict(pos=FAKE, top_k=128, pstride=64), b"multiple"), (dict(q=None), b"null"), (dict(out=None), b"null"),
    (dict(q=ctypes.c_void_p(4104)), b"aligned"), (dict(qst=4100), b"aligned"), (dict(bytes=64), b"workspace"),
    (dict(bs=1 << 20, tcols=1 << 24, tstride=1 << 24), b"units"), (dict(planned=1, pos=FAKE, top_k=128, pstride=128), b"whole")])
def test_decode_refuses(lib, kw, said):
    a = dict(q=FAKE, qd=0, qst=4096, H=32, kn=None, vn=None, nd=0, loc=None, **CACHE, table=FAKE, tstride=4, trows=2, tcols=4,
             rpi=FAKE, seq=FAKE, bs=2, pos=None, pstride=0, top_k=0, scale=0.1, out=FAKE, ws=FAKE, bytes=1 << 30,
             planned=0)
    a.update(kw)
    refused(lib.qq_fp8_decode_attention(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", [
    (dict(blocks=0), b"blocks"), (dict(kv=0), b"KV heads"), (dict(dim=80), b"head_dim"), (dict(trows=0), b"bad sizes"),
    (dict(tcols=0), b"bad sizes"), (dict(bs=-1), b"bad sizes"), (dict(rpi=None), b"null"), (dict(seq=None), b"null"),
    (dict(ws=None), b"null"), (dict(bytes=64), b"workspace"), (dict(bs=1 << 20, tcols=1 << 24), b"units")])
def test_decode_plan_refuses(lib, kw, said):
    a = dict(blocks=5, kv=4, dim=128, trows=2, tcols=4, rpi=FAKE, seq=FAKE, bs=2, ws=FAKE, bytes=1 << 30)
    a.update(kw)
    refused(lib.qq_fp8_decode_plan(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [
    (dict(phase=0), b"phase"), (dict(phase=4), b"phase"), (dict(bounds=None), b"null"), (dict(scores=None), b"null"),
    (dict(pos=None), b"null"), (dict(limit=None), b"null"), (dict(layer=-1), b"bad sizes"), (dict(reqs=0), b"bad sizes"),
    (dict(top_k=100), b"multiple"), (dict(top_k=64 * 1026), b"selected pages"), (dict(kv=16, H=32), b"exceeds"),
    (dict(loc=None), b"null"), (dict(nd=7), b"dtype"), (dict(kn=ctypes.c_void_p(4104)), b"aligned"), (dict(bytes=64), b"workspace")])
def test_quest_step_refuses(lib, kw, said):
    a = dict(q=FAKE, qd=0, qst=4096, H=32, kn=FAKE, vn=FAKE, nd=0, loc=FAKE, **CACHE, table=FAKE, tstride=4, trows=2, tcols=4,
             bounds=FAKE, layer=0, rpi=FAKE, seq=FAKE, limit=FAKE, bs=2, reqs=2, mp=4, top_k=128, scale=0.1, scores=FAKE, pos=FAKE,
             out=FAKE, ws=FAKE, bytes=1 << 30, phase=3, planned=0)
    a.update(kw)
    refused(lib.qq_fp8_quest_step(*a.values(), None), lib, said)


@pytest.mark.parametrize("kw, said", BAD_CACHE + [
    (dict(H=30), b"divisible"), (dict(scale=0.0), b"positive"), (dict(scale=float("nan")), b"positive"),
    (dict(scale=float("inf")), b"positive"), (dict(bs=-1), b"bad sizes"), (dict(n=1 << 28), b"bad sizes"),
    (dict(tstride=3), b"bad sizes"), (dict(q=None), b"null"), (dict(ext=None), b"null"), (dict(out=ctypes.c_void_p(4104)), b"aligned"),
    (dict(n=8, tcols=1 << 12, tstride=1 << 12, ws=None), b"workspace")])
def test_extend_refuses(lib, kw, said):
    a = dict(q=FAKE, H=32, **CACHE, table=FAKE, tstride=4, trows=2, tcols=4, rpi=FAKE, seq=FAKE, prefix=FAKE, ext=FAKE, bs=2, n=10,
             scale=0.1, out=FAKE, ws=FAKE, bytes=1 << 30)
    a.update(kw)
    refused(lib.qq_fp8_extend_attention(*a.values(), None), lib, said)


def test_decode_workspace(lib):
    assert lib.qq_fp8_decode_workspace_bytes(0, 32, 4, 128) == 0
    assert lib.qq_fp8_decode_workspace_bytes(2, 30, 4, 128) == 0
    small, large = (lib.qq_fp8_decode_workspace_bytes(bs, 32, 4, 128) for bs in (1, 1000))
    assert 0 < small < large < 32 << 20


def test_a_plan_is_its_capture_s(monkeypatch):
    """A plan made in one graph capture, or in none, is of no use in another."""
    ids = {11: 0, 12: 5}
    monkeypatch.setattr(_lib, "capture_id", lambda device, stream: ids[stream])
    ws = torch.empty(1)
    eager, captured, unsaid = (DecodePlan(2, ws, s, i) for s, i in ((11, 0), (12, 5), (12, -1)))
    assert eager.usable(11) and captured.usable(12) and not eager.usable(12) and not captured.usable(11)
    ids.update({11: 6, 12: 6})  # two other captures on those streams
    assert not eager.usable(11) and not captured.usable(12)
    ids[12] = 0
    assert not captured.usable(12)
    ids[12] = -1  # the runtime does not say
    assert not unsaid.usable(12)


# ---------------------------------------------------------------- the division of the work


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    cxx = shutil.which("g++") or "/opt/rocm/llvm/bin/clang++"
    d = tmp_path_factory.mktemp("fp8rules")
    (d / "shim.cpp").write_text("""
#include "qq_rules.h"
using namespace qq::rules;
extern "C" int64_t slices_(int64_t heads) { return fp8_max_slices((int)heads); }
extern "C" int64_t len_(int64_t total, int64_t longest, int64_t most) { return fp8_slice_len(total, longest, most); }
extern "C" int64_t parts_() { return kFp8Parts; }
""")
    out = str(d / "lib.so")
    subprocess.run([cxx, "-std=c++17", "-O1", "-fPIC", "-shared", "-Wall", "-Werror", f"-I{CSRC}", "-o", out, str(d / "shim.cpp")],
                   check=True)
    lib = ctypes.CDLL(out)
    for f in (lib.slices_, lib.len_, lib.parts_):
        f.restype = ctypes.c_int64
    lib.slices_.argtypes = [ctypes.c_int64]
    lib.len_.argtypes = [ctypes.c_int64] * 3
    return lib


def test_slices_cover_the_batch_within_the_grid_and_the_merge(rules):
    rng = random.Random(1)
    for _ in range(2000):
        heads = rng.choice([1, 2, 3, 4, 8, 12, 64, 600])
        units = [rng.choice([1, 2, 33, rng.randint(1, 5000), 1 << 20]) for _ in range(rng.choice([1, 2, 7, 100, 700]))]
        total, most = sum(units), rules.slices_(heads)
        n = rules.len_(total, max(units), most)
        slices = -(-total // n)
        assert 1 <= slices <= most and (heads * most <= 256 or most == 1)  # a block per CU
        at = 0
        for u in units:  # parts of a request
            assert (at + u - 1) // n - at // n + 1 <= rules.parts_()
            at += u


# ---------------------------------------------------------------- the oracle itself


def test_oracle_rounds_as_torch_does():
    y = torch.linspace(-448, 448, 100001, dtype=torch.float64)
    y = torch.cat([y, y * 2.0**-10, y * 2.0**-17])
    want = y.to(torch.float32).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(of.round_e4m3(y.float().double().numpy()), want)


def test_oracle_scales():
    assert of.exponent(0.0) == -110 and of.exponent(1e-40) == -110
    assert of.exponent(448.0) == 0 and of.exponent(np.nextafter(448.0, 500)) == 1 and of.exponent(224.0) == -1
    c = of.Cache(3, 1, 2)
    c.write([64], np.array([[[1.0, 2.0]]]), np.array([[[0.1, 0.0]]]))
    c.write([65], np.array([[[448.0 * 8, 0.0]]]), np.array([[[np.inf, 1.0]]]))
    k, v = c.rows([64, 65])
    assert k[0, 0].tolist() == [1.0, 2.0] and k[1, 0].tolist() == [3584.0, 0.0]
    assert np.isnan(v).all() and np.isnan(c.scale(1)[1]).all() and c.scale(0)[1, 0] == 8.0
