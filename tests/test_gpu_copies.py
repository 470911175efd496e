"""Copies and pickles of what keeps addresses of its own tensors: they work on their own memory."""

from __future__ import annotations

import copy
import io
import pickle

import pytest
import torch

from qwenquest_amd import QKNormRotary
from qwenquest_amd.paged import BlockReqToTokenPool, Fp4TokenToKVPool, Fp8TokenToKVPool

pytestmark = pytest.mark.gpu


def saved(x):
    buf = io.BytesIO()
    torch.save(x, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


COPIES = {"deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x)), "saved": saved}


@pytest.mark.parametrize("how", COPIES)
def test_rotations(cuda, how):
    gen = torch.Generator(device=cuda).manual_seed(0)
    wq, wk = (torch.empty(64, device=cuda).uniform_(0.5, 2.0, generator=gen) for _ in range(2))
    op = QKNormRotary(4, 2, 64, q_weight=wq, k_weight=wk, sections=(10, 22), base=1e5, device=cuda)
    x, pos = torch.randn(30, 512, device=cuda), torch.randint(0, 5000, (2, 30), device=cuda)
    want = op(x, pos)
    other = COPIES[how](op)
    for t in (*op._weights, op._quarters, op._axis):
        t.zero_()
    assert all(torch.equal(a, b) for a, b in zip(other(x, pos), want))
    assert not torch.equal(op(x, pos)[0], want[0])
    again = copy.copy(other)
    assert all(torch.equal(a, b) for a, b in zip(again(x, pos), want))


@pytest.mark.parametrize("how", COPIES)
@pytest.mark.parametrize("kind", [Fp4TokenToKVPool, Fp8TokenToKVPool])
def test_pools(cuda, kind, how):
    pool = kind(6, 2, 2, 64, cuda)
    loc = torch.arange(64, 264, device=cuda)
    k, v, other_k = (torch.randn(200, 2, 64, device=cuda) for _ in range(3))
    pool.set_kv_buffer(1, loc, k, v)
    want = pool.get_rows(1, loc)
    other = COPIES[how](pool)
    assert all(torch.equal(a, b) for a, b in zip(other.get_rows(1, loc), want))
    other.set_kv_buffer(1, loc, other_k, v)  # of its own
    assert all(torch.equal(a, b) for a, b in zip(pool.get_rows(1, loc), want))
    pool.set_kv_buffer(1, loc, v, k)
    assert not torch.equal(other.get_rows(1, loc)[0], pool.get_rows(1, loc)[0])
    assert torch.equal(other.get_rows(1, loc)[1], want[1])


@pytest.mark.parametrize("how", COPIES)
def test_request_pools(cuda, how):
    pool = BlockReqToTokenPool(3, 400, 12, cuda)
    i64 = lambda *x: torch.tensor(x, device=cuda)  # noqa: E731
    pool.assign(i64(0, 1), i64(0, 0), i64(100, 70), 170)
    other = COPIES[how](pool)
    for x in (pool, other):
        assert x.available_blocks() == 7 and x.held.tolist() == [2, 2, 0]
    loc, pos = other.assign(i64(2), i64(0), i64(200), 200)
    assert other.available_blocks() == 3 and other.held.tolist() == [2, 2, 4] and pos.tolist() == list(range(200))
    assert torch.equal(other.req_to_token[2, :200].long(), loc) and (loc > 0).all()
    assert pool.available_blocks() == 7 and pool.held.tolist() == [2, 2, 0] and not pool.block_table[2].any()
    pool.release(i64(0))
    assert pool.available_blocks() == 9 and other.available_blocks() == 3 and other.block_table[0, 0] > 0
    other.assign(i64(0), i64(100), i64(301), 301)  # past its table
    pool.check_errors()
    torch.cuda.synchronize()
    with pytest.raises(ValueError):
        other.poll_errors()
    pool.poll_errors()
