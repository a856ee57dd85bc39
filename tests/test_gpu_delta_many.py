"""Gated delta rule (include/kmamba_delta.h) with many sequences: more blocks than the device has SMs, so that a block takes
two units of 16 columns (the second one of an odd count lies past dv); short and long packed sequences, more of them than
are sorted by length.  Against the definition in 64 bits with its derivative by autograd, all sequences at once."""
import random

import pytest
import torch

import mixer_ref as ref
from test_gpu_delta import _compare, _inputs, _run

pytestmark = pytest.mark.gpu


def _definition(q, k, v, g, beta, h0, scale):
    """q, k [N, T, Hv, dk], v [N, T, Hv, dv], g, beta [N, T, Hv], h0 [N, Hv, dk, dv]"""
    S, out = h0, []
    for t in range(q.shape[1]):
        S = torch.exp(g[:, t])[..., None, None] * S
        u = beta[:, t][..., None] * (v[:, t] - torch.einsum("nhk,nhkv->nhv", k[:, t], S))
        S = S + torch.einsum("nhk,nhv->nhkv", k[:, t], u)
        out.append(scale * torch.einsum("nhk,nhkv->nhv", q[:, t], S))
    return torch.stack(out, 1), S


def _want(x, dev, cu=None, scale=0.5):
    """Results and gradients on the device.  Packed sequences are laid out one per row; a place behind a sequence's end has
    no key, no strength and no decay, and so changes nothing."""
    B, T, Hk, dk = x["q"].shape
    Hv = x["v"].shape[2]
    cu = [b * T for b in range(B + 1)] if cu is None else cu
    n = len(cu) - 1
    longest = max(b - a for a, b in zip(cu, cu[1:]))
    at = torch.full((n, longest), B * T)
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        at[i, :b - a] = torch.arange(a, b)
    leaf = {m: x[m].to(dev).double().requires_grad_(True) for m in ("q", "k", "v", "g", "beta", "h0")}

    def rows(t, heads):
        flat = t.reshape((B * T,) + t.shape[2:])
        t = torch.cat([flat, torch.zeros_like(flat[:1])])[at.to(dev)]
        return t.repeat_interleave(Hv // heads, 2) if heads != Hv else t

    o, hT = _definition(rows(leaf["q"], Hk), rows(leaf["k"], Hk), rows(leaf["v"], Hv), rows(leaf["g"], Hv),
                        rows(leaf["beta"], Hv), leaf["h0"], scale)
    back = torch.empty(B * T, dtype=torch.long)
    places = at.flatten()
    inside = places < B * T
    back[places[inside]] = torch.arange(places.numel())[inside]
    o = o.flatten(0, 1)[back.to(dev)].reshape(x["v"].shape)
    got = torch.autograd.grad([o, hT], list(leaf.values()), [x["do"].to(dev).double(), x["dhT"].to(dev).double()])
    res = {"o": o.detach(), "hT": hT.detach()}
    res.update(("d" + m, t) for m, t in zip(leaf, got))
    return res


# (B, T, Hk, Hv, dk, dv): every count of sequences x heads x units is above the SMs of any device of this kind (148 to
# 160); 3 units: the second block's second unit is empty; 200 tokens: more chunks than stages
SHAPES = [(40, 140, 1, 2, 64, 48), (30, 200, 2, 2, 60, 64), (40, 65, 2, 2, 128, 48), (12, 200, 1, 2, 128, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_more_units_than_sms(kmb, cuda, shape, dtype):
    x = _inputs(*shape, dtype, seed=sum(shape))
    _compare(_run(kmb, cuda, x), _want(x, cuda), dtype)
    fwd = _run(kmb, cuda, x, backward=False)
    both = _run(kmb, cuda, x)
    assert torch.equal(fwd["o"], both["o"]) and torch.equal(fwd["hT"], both["hT"])


def _offsets(n, T, seed):
    """n lengths of 0 to 6 tokens and a few long ones, T tokens in all."""
    r = random.Random(seed)
    lens = [r.randint(0, 6) for _ in range(n)]
    for i in (n // 3, n // 2, n - 1):
        lens[i] = r.randint(100, 160)
    lens[7] += T - sum(lens)
    assert min(lens) >= 0
    cu = [0]
    for m in lens:
        cu.append(cu[-1] + m)
    return cu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,T,Hk,Hv,dk,dv", [(300, 1500, 2, 4, 64, 48), (700, 2900, 1, 2, 64, 32), (520, 2300, 2, 4, 128, 48),
                                             (513, 2300, 1, 1, 32, 16)])
def test_many_packed_sequences(kmb, cuda, n, T, Hk, Hv, dk, dv, dtype):
    """Above and below 512 sequences, and with more units than a block each would fill the device several times."""
    cu = _offsets(n, T, n)
    x = _inputs(1, T, Hk, Hv, dk, dv, dtype, seed=n, seqs=n)
    _compare(_run(kmb, cuda, x, cu=cu), _want(x, cuda, cu=cu), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("packed", [False, True])
def test_a_sequence_does_not_depend_on_the_others(kmb, cuda, packed, dtype):
    """The same bits alone and among so many that blocks take two units."""
    n, T, Hk, Hv, dk, dv = 100, 70, 1, 2, 64, 80   # 1000 units
    x = _inputs(1 if packed else n, T * n if packed else T, Hk, Hv, dk, dv, dtype, seed=5, seqs=n)
    few = {m: t[:2] if not packed or m in ("h0", "dhT") else t[:, :2 * T].contiguous() for m, t in x.items()}
    cu = [T * i for i in range(n + 1)] if packed else None
    many, two = _run(kmb, cuda, x, cu=cu), _run(kmb, cuda, few, cu=None if cu is None else cu[:3])
    for m in two:
        part = many[m][:2] if not packed or m in ("hT", "dh0") else many[m][:, :2 * T]
        assert torch.equal(part, two[m]), m
