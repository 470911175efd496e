"""Operators that fill their outputs behind torch's back, through the C entries, refuse torch.jit.trace: a trace would
keep their allocations alone.  No GPU: they refuse before anything else."""

from __future__ import annotations

import pytest
import torch

from qwenquest_amd import QKNormRotary

X = torch.zeros(2, 4)


def refused(f):
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, X, check_trace=False)


def test_rotation():
    op = object.__new__(QKNormRotary)
    refused(lambda x: op(x, X))
    refused(lambda x: op.apply(x, x, X))
