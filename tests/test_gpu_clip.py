"""Global gradient norm and clipping (include/kmamba_clip.h) against 64 bits.  The sum is kept in 64 bits over fp32
partial sums of 16 to 32 squares: the norm is within 8 units of 2^-24, a clipped entry within the coefficient's and
its own rounding."""
import ctypes as C
import math

import pytest
import torch

import mixer_ref as ref

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


def _clip(kmb, grads, max_norm, outs=None):
    lst = kmb.grad_list(grads, outs)
    ws = torch.full((kmb.grad_clip_workspace_floats(lst),), float("nan"), device="cuda")
    res = torch.full((2,), float("nan"), device="cuda")
    kmb.grad_clip(lst, max_norm, res, ws)
    torch.cuda.synchronize()
    return [float(v) for v in res.cpu()]


def _tensors(sizes, seed=0, odd=True, scale=1.0, mixed=True):
    """Views at odd places of larger buffers."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = torch.bfloat16 if mixed and i % 2 else torch.float32
        big = (torch.randn(n + 9, generator=gen) * scale).to(dt).cuda()
        out.append(big[(i % 9 if odd else 0):][:n])
    return out


SIZES = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 64, 0, 1000, 4097, 8192, 8193, 16385, 100003]


@pytest.mark.parametrize("place", ["in_place", "apart", "apart_unaligned"])
@pytest.mark.parametrize("ratio", [0.1, 0.999, 3.0])
def test_clip(kmb, cuda, place, ratio):
    grads = _tensors(SIZES)
    before = [g.clone() for g in grads]
    norm, _ = ref.clip([g.cpu() for g in before], 1.0)
    max_norm = norm * ratio
    outs = None
    if place != "in_place":
        shift = 0 if place == "apart" else 1
        outs = [torch.full((g.numel() + 1,), float("nan"), dtype=g.dtype, device=cuda)[shift:shift + g.numel()]
                for g in grads]
    got, coef = _clip(kmb, grads, max_norm, outs)
    assert abs(got - norm) <= 8 * UNIT * norm
    want = min(1.0, max_norm / norm)
    assert abs(coef - want) <= 8 * UNIT
    if outs is not None:
        for g, b in zip(grads, before):
            assert torch.equal(g, b)
    for o, b in zip(grads if outs is None else outs, before):
        if coef == 1.0:
            assert torch.equal(o, b)
        else:
            assert torch.equal(o, (b.float() * coef).to(b.dtype))


@pytest.mark.parametrize("n", [1, 63, 64, 65, 255, 256, 257, 700])
def test_many_tensors(kmb, cuda, n):
    grads = _tensors([(i * 37) % 301 for i in range(n)], seed=n)
    norm, coef = ref.clip([g.cpu() for g in grads], 0.5)
    before = [g.clone() for g in grads]
    got, c = _clip(kmb, grads, 0.5)
    assert abs(got - norm) <= 8 * UNIT * max(norm, 1e-30) and abs(c - coef) <= 8 * UNIT
    for g, b in zip(grads, before):
        assert torch.equal(g, (b.float() * c).to(b.dtype))


@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e25, 1e-22])
def test_squares_outside_fp32(kmb, cuda, scale):
    grads = _tensors([5000, 3, 77, 1], scale=scale, seed=4)
    norm, _ = ref.clip([g.cpu() for g in grads], 1.0)
    got, coef = _clip(kmb, grads, norm * 0.5)
    assert abs(got - norm) <= 8 * UNIT * norm and abs(coef - 0.5) <= 8 * UNIT


def test_large_and_small_together(kmb, cuda):
    """One huge entry among ones, zeros, subnormals."""
    a = torch.ones(100000, device=cuda)
    a[77777] = 1e20
    norm, _ = ref.clip([a.cpu()], 1.0)
    got, _ = _clip(kmb, [a], math.inf)
    assert abs(got - norm) <= 8 * UNIT * norm
    z = torch.zeros(4096, device=cuda)
    assert _clip(kmb, [z], 1.0) == [0.0, 1.0]
    s = torch.full((64,), 1e-40, device=cuda)
    got, _ = _clip(kmb, [s], 1.0)
    assert abs(got - float(s.cpu().double().norm())) <= 8 * 2.0 ** -149


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_not_finite(kmb, cuda, bad):
    """The gradients stay as they are, in place and apart, and the norm says so."""
    g = torch.randn(3000, device=cuda)
    g[1234] = bad
    before = g.clone()
    out = torch.zeros_like(g)
    got, coef = _clip(kmb, [g], 1.0, [out])
    assert not math.isfinite(got) and coef == 1.0
    assert torch.equal(out.view(torch.int32), before.view(torch.int32))
    _clip(kmb, [g], 1.0)
    assert torch.equal(g.view(torch.int32), before.view(torch.int32))


def test_measured_only_and_empty(kmb, cuda):
    grads = _tensors([100, 200], seed=9)
    before = [g.clone() for g in grads]
    norm, _ = ref.clip([g.cpu() for g in grads], 1.0)
    got, coef = _clip(kmb, grads, 1e-3, [None, None])
    assert abs(got - norm) <= 8 * UNIT * norm and coef < 1.0
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert _clip(kmb, [], 1.0) == [0.0, 1.0]
    assert _clip(kmb, [torch.empty(0, device=cuda)], 1.0) == [0.0, 1.0]


def test_same_bits_every_time(kmb, cuda):
    grads = _tensors([3_000_001, 77], seed=3, mixed=False)
    a = _clip(kmb, [g.clone() for g in grads], 2.0)
    assert a == _clip(kmb, [g.clone() for g in grads], 2.0)


def test_model_arena(kmb, cuda):
    """Between the model's backward and its AdamW step; clip_norm of the optimizer's config is the default bound."""
    import numpy as np
    cfg = kmb.model_config([32], 64, 32, 8, 1, 2)
    L = kmb.lib()
    m = L.kmamba_create(C.byref(cfg))
    assert m, kmb.last_error()
    assert L.kmamba_init(m, 1) == 0
    opt = kmb.MBOptimConfig()
    L.kmamba_optim_config_set_defaults(C.byref(opt))
    opt.clip_norm = 0.125
    res, ws = torch.zeros(2, device=cuda), torch.zeros(L.kmb_grad_clip_workspace_floats(1), device=cuda)
    assert L.kmb_model_clip_gradients(m, 0.0, res.data_ptr(), ws.data_ptr(), None) == -1   # no optimizer yet
    assert L.kmamba_enable_training(m, C.byref(opt), 1e-3, 0.0) == 0
    tok = torch.randint(0, 64, (2, 33), dtype=torch.int32, device=cuda)
    loss = L.kmb_model_forward_backward(m, tok.data_ptr(), 2, None)
    assert np.isfinite(loss)
    n = C.c_size_t()
    ptr = L.kmb_model_grad_arena(m, C.byref(n))
    arena = torch.as_tensor(kmb.DeviceArray(ptr, n.value), device=cuda)
    before = arena.clone()
    want = float(before.double().norm())
    assert want > 0.125
    kmb.check(L.kmb_model_clip_gradients(m, 0.0, res.data_ptr(), ws.data_ptr(), None), "kmb_model_clip_gradients")
    torch.cuda.synchronize()
    norm, coef = (float(v) for v in res.cpu())
    assert abs(norm - want) <= 8 * UNIT * want and abs(coef - 0.125 / want) <= 8 * UNIT
    assert torch.equal(arena, before * coef)
    assert L.kmb_model_optimizer_step(m, None) == 0
    torch.cuda.synchronize()
    L.kmamba_free(m)
