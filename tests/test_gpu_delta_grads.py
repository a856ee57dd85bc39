"""Gated delta rule (include/kmamba_delta.h): gradients where the products behind them are short, and per token."""
import math

import pytest
import torch

import mixer_ref as ref
from test_gpu_delta import _compare, _inputs, _reference, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("dv", [1, 16, 64])
def test_few_columns_and_shared_heads(kmb, cuda, dv, dk, dtype):
    """One slice of dv or less: nothing but its own barrier orders a head's decay tables, and the next head of the block
    writes them again.  Right, and the same bits every time."""
    x = _inputs(2, 150, 2, 6, dk, dv, dtype, seed=dk + dv)
    x["g"] = x["g"] * torch.tensor([0.01, 1.0, 10.0]).repeat(2)   # neighbouring heads' tables differ
    first = _run(kmb, cuda, x)
    _compare(first, _reference(x), dtype)
    for _ in range(10):
        again = _run(kmb, cuda, x)
        for n in first:
            assert torch.equal(first[n], again[n]), n
