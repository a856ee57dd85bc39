"""Gated delta rule (include/kmamba_delta.h): bf16 results are the fp32 ones rounded once.

A result whose error before the rounding is e (2-norm, at most 4e-6 of the result, as in the tests of fp32) differs from
the rounded definition where an entry's error crosses a rounding boundary: with a probability of at most 2 |e_i| over
the spacing of bf16, which is at most 2^-7 |x_i|, and then by that spacing.  So the squared difference is about
sum 2 |e_i| 2^-7 |x_i| <= 2^-6 |e| |x|: at most sqrt(2^-6 4e-6) = 2.5e-4 of the result."""
import math

import pytest
import torch

import mixer_ref as ref
from test_gpu_delta import F32, _inputs, _reference, _run

pytestmark = pytest.mark.gpu
ONCE = math.sqrt(2.0 ** -6 * F32)

# (B, T, Hk, Hv, dk, dv): both widths of the key tiles, whole and odd chunks, shared key heads
SHAPES = [(1, 200, 1, 2, 64, 64), (2, 130, 1, 1, 128, 128), (1, 192, 2, 2, 100, 48)]


def _once(got, want):
    return ref.rel(got, want.to(torch.bfloat16))


@pytest.mark.parametrize("shape", SHAPES)
def test_outputs_are_rounded_once(kmb, cuda, shape):
    x = _inputs(*shape, torch.bfloat16, seed=sum(shape))
    got, want = _run(kmb, cuda, x, backward=False), _reference(x, backward=False)
    assert _once(got["o"], want["o"]) <= ONCE


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_keeping_for_the_backward_changes_no_bit(kmb, cuda, shape, dtype):
    x = {n: t.to(cuda) for n, t in _inputs(*shape, dtype, seed=sum(shape)).items()}
    outs = []
    for keep in (False, True):
        o, hT = torch.empty_like(x["v"]), torch.empty_like(x["h0"])
        p = kmb.delta_params(x["q"], x["k"], x["v"], x["g"], x["beta"], o, scale=0.5, h0=x["h0"], hT=hT)
        kmb.delta_forward(p, torch.empty(kmb.delta_workspace_floats(p, keep), device=cuda), keep=keep)
        outs.append((o, hT))
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_are_rounded_once(kmb, cuda, shape):
    x = _inputs(*shape, torch.bfloat16, seed=sum(shape) + 1)
    got, want = _run(kmb, cuda, x), _reference(x)
    for n in ("o", "dq", "dk", "dv"):
        assert _once(got[n], want[n]) <= ONCE, n
