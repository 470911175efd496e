"""Calls past what a launch holds, 2^32 threads: refused before anything is launched.  No GPU."""

from __future__ import annotations

import pytest

from tests.test_block_pools import CACHE, FAKE, lib, refused  # noqa: F401 - lib: a fixture

MOST = (1 << 24) - 1  # blocks of 256 threads
LARGE = 1 << 60  # bytes of a workspace


def decode(lib, kind, planned, **kw):  # noqa: F811
    a = dict(q=FAKE, qd=0, qst=128, H=1, kn=FAKE, vn=FAKE, nd=0, loc=FAKE, **{**CACHE, "kv": 1, "dim": 128}, table=FAKE, tstride=1, trows=2, tcols=1,
             rpi=FAKE, seq=FAKE, bs=2, pos=None, pstride=0, top_k=0, scale=0.1, out=FAKE, ws=FAKE, bytes=LARGE, planned=planned)
    a.update(kw)
    return getattr(lib, f"qq_{kind}_decode_attention")(*a.values(), None)


# a block for the plan, one for each request whose pages are selected, and the new tokens': of 8 bits two each, of 4 bits one
# for 1024 / dim
@pytest.mark.parametrize("kind, bs, kv, dim", [("fp4", MOST, 1, 128), ("fp4", 1 << 25, 1, 64), ("fp4", 1 << 20, 200, 128),
                                               ("fp8", 1 << 23, 1, 128), ("fp8", 1 << 13, 1024, 64)])
def test_decode_batches_past_a_launch(lib, kind, bs, kv, dim):  # noqa: F811
    refused(decode(lib, kind, 0, bs=bs, kv=kv, H=kv, dim=dim, qst=kv * dim), lib, b"bad sizes")


@pytest.mark.parametrize("kind, bs, kv", [("fp4", MOST, 1), ("fp4", 1 << 23, 8), ("fp8", 1 << 23, 1)])
def test_quest_steps_past_a_launch(lib, kind, bs, kv):  # noqa: F811
    for phase in (2, 3):
        a = dict(q=FAKE, qd=0, qst=4096, H=kv, kn=FAKE, vn=FAKE, nd=0, loc=FAKE, **{**CACHE, "kv": kv}, table=FAKE, tstride=1, trows=2, tcols=1,
                 bounds=FAKE, layer=0, rpi=FAKE, seq=FAKE, limit=FAKE, bs=bs, reqs=2, mp=4, top_k=128, scale=0.1, scores=FAKE, pos=FAKE,
                 out=FAKE, ws=FAKE, bytes=LARGE, phase=phase, planned=0)
        refused(getattr(lib, f"qq_{kind}_quest_step")(*a.values(), None), lib, b"bad sizes")


def test_a_prefill_past_a_launch(lib):  # noqa: F811
    a = dict(q=FAKE, H=1, **{**CACHE, "kv": 1, "dim": 64}, table=FAKE, tstride=1, trows=2, tcols=1, rpi=FAKE, seq=FAKE, prefix=FAKE, ext=FAKE,
             bs=MOST, n=1, scale=0.1, out=FAKE, ws=FAKE, bytes=LARGE)
    refused(lib.qq_fp4_extend_attention(*a.values(), None), lib, b"too many query rows")
