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


@pytest.mark.parametrize("shape", [(1, 140, 1, 2, 64, 48), (1, 140, 1, 1, 128, 80)])
@pytest.mark.parametrize("at", [3, 67])
def test_a_large_gradient_costs_its_own_block_only(kmb, cuda, at, shape):
    """do at one token is 1e9 times the others'.  What the tokens of later blocks of 16 get does not depend on it and is as
    accurate as without it."""
    x = _inputs(*shape, torch.float32, seed=17)
    x["do"][0, at] *= 1e9
    got, want = _run(kmb, cuda, x), _reference(x)
    rest = slice((at | 15) + 1, None)
    for n in ("dq", "dk", "dv", "dbeta"):
        bound = 1e-5 if n == "dbeta" else 4e-6
        assert ref.rel(got[n][:, rest], want[n][:, rest]) <= bound, n
    before = slice(0, at & ~15)   # dq needs nothing but its own token's do
    if at > 15:
        assert ref.rel(got["dq"][:, before], want["dq"][:, before]) <= 4e-6


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_that_are_not_finite(kmb, cuda, dtype, bad):
    """One at token 70, column 3 of do: the other head, later blocks of 16 tokens, and the queries of every other block
    keep their bits."""
    x = _inputs(1, 140, 2, 2, 64, 48, dtype, seed=19)
    clean = _run(kmb, cuda, x)
    x["do"][0, 70, 0, 3] = bad
    got = _run(kmb, cuda, x)
    for n in ("dq", "dk", "dv", "dg", "dbeta"):
        assert torch.equal(got[n][0, :, 1], clean[n][0, :, 1]), n
    for n in ("dq", "dk", "dv", "dbeta"):
        assert torch.equal(got[n][0, 80:, 0], clean[n][0, 80:, 0]), n
    assert torch.equal(got["dg"][0, 128:, 0], clean["dg"][0, 128:, 0])
    assert torch.equal(got["dq"][0, :64, 0], clean["dq"][0, :64, 0])
    assert not torch.isfinite(got["dq"][0, 70, 0]).any()
