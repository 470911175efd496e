"""Operators that fill their outputs behind torch's back, through the C entries, refuse torch.jit.trace: a trace would
keep their allocations alone.  No GPU: they refuse before anything else."""

from __future__ import annotations

import pytest
import torch

from qwenquest_amd import QKNormRotary, QuestAlgorithm
from qwenquest_amd.attention import ops
from qwenquest_amd.paged import Fp4TokenToKVPool, Fp8TokenToKVPool

X = torch.zeros(2, 4)


def refused(f):
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, X, check_trace=False)


def test_rotation():
    op = object.__new__(QKNormRotary)
    refused(lambda x: op(x, X))
    refused(lambda x: op.apply(x, x, X))


@pytest.mark.parametrize("kind", [Fp4TokenToKVPool, Fp8TokenToKVPool])
def test_pools_of_codes(kind):
    pool = object.__new__(kind)
    refused(lambda x: pool.get_rows(0, x))
    refused(lambda x: (pool.set_kv_buffer(0, X, x, x), x)[1])
    refused(lambda x: ops.coded_decode_plan(pool, X, X, x).workspace)
    refused(lambda x: ops.coded_decode_attention(x, pool, 0, X, X, X, 0.1))
    refused(lambda x: ops.coded_quest_step(x, x, x, X, pool, 0, X, None, X, X, 0.1))
    refused(lambda x: ops.coded_extend_attention(x, pool, 0, X, X, X, X, X, 0.1))
    quest = object.__new__(QuestAlgorithm)
    refused(lambda x: (quest.update_prefill_representations_blocks(X, x, pool, X), x)[1])
    refused(lambda x: (quest.decode_step_blocks(X, x, pool, X), x)[1])
