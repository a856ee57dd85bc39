"""Gated delta rule (include/kmamba_delta.h): g = -inf forgets the state, whatever is in it (an entry of a pool that
nobody has written, say)."""
import math

import pytest
import torch

import mixer_ref as ref
from test_gpu_delta import BF16, F32, _compare, _inputs, _reference, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(kmb, cuda, dtype, bad):
    x = _inputs(2, 2, 1, 2, 100, 37, dtype, seed=3)
    x["g"][:, 0] = -math.inf
    pool = torch.full((2, 2, 100, 37), bad, device=cuda)
    d = {n: x[n].to(cuda) for n in ("q", "k", "v", "g", "beta")}
    o = torch.empty_like(d["v"])
    kmb.delta_step(kmb.delta_params(d["q"], d["k"], d["v"], d["g"], d["beta"], o), pool)
    torch.cuda.synchronize()
    want, S = ref.delta(x["q"], x["k"], x["v"], x["g"], x["beta"], None, 1.0)
    assert ref.rel(o, want) <= (BF16 if dtype == torch.bfloat16 else F32)
    assert ref.rel(pool, S) <= F32


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 130, 1, 2, 64, 48), (1, 70, 1, 1, 128, 80)])
def test_first_token(kmb, cuda, shape, dtype, bad):
    """The chunked form and its gradients, from an initial state that holds the value in one place or everywhere."""
    x = _inputs(*shape, dtype, seed=5)
    x["g"][:, 0] = -math.inf
    want = _reference(dict(x, h0=torch.zeros_like(x["h0"])))
    want["dg"] = torch.nan_to_num(want["dg"])
    for where in (slice(None), (0, 0, 7, 5)):
        x["h0"][where] = bad
        got = _run(kmb, cuda, x)
        _compare(got, want, dtype)
        assert float(got["dh0"].abs().max()) == 0.0

