"""Refusals of the mixer's operators: each invalid argument returns -1 with a reason, before anything reaches a device
(no GPU is needed).  And the 64-bit forms of the tests themselves, against differences."""
import ctypes as C
import math

import pytest
import torch

import mixer_ref as ref


def _delta(kmb, **kw):
    p = kmb.KMBDeltaParams()
    p.batch, p.T, p.Hk, p.Hv, p.dk, p.dv, p.dtype, p.scale = 1, 8, 1, 2, 16, 16, 1, 1.0
    p.q = p.k = p.v = p.o = 4096
    for k, v in kw.items():
        setattr(p, k, v)
    return p


BAD_DELTA = [dict(batch=-1), dict(T=-1), dict(Hk=0), dict(Hv=0), dict(Hk=2, Hv=3), dict(dk=0), dict(dv=0),
             dict(dk=129), dict(dv=129), dict(dtype=2), dict(cu_seqlens=4096, n_seq=0),
             dict(cu_seqlens=4096, n_seq=1, batch=2), dict(ld_q=15), dict(ld_k=1), dict(ld_v=31), dict(ld_o=31),
             dict(batch=70000, T=70000), dict(ld_q=1 << 31), dict(q=None), dict(k=None), dict(v=None), dict(o=None)]


@pytest.mark.parametrize("bad", BAD_DELTA, ids=[str(b) for b in BAD_DELTA])
def test_delta_refusals(kmb, bad):
    L, p = kmb.lib(), _delta(kmb, **bad)
    assert L.kmb_delta_forward(C.byref(p), 4096, 0, None) == -1
    assert kmb.last_error().startswith("delta")
    if not any(bad.get(n, 0) is None for n in ("q", "k", "v", "o")):
        assert L.kmb_delta_workspace_floats(C.byref(p), 1) == 0
    if "cu_seqlens" not in bad:
        assert L.kmb_delta_step(C.byref(p), 4096, 4, None, None) == -1
        assert "delta" in kmb.last_error()


def test_delta_more_refusals(kmb):
    L, p = kmb.lib(), _delta(kmb)
    assert L.kmb_delta_forward(None, 4096, 0, None) == -1
    assert L.kmb_delta_forward(C.byref(p), None, 0, None) == -1 and "workspace" in kmb.last_error()
    assert L.kmb_delta_forward(C.byref(p), 4100, 0, None) == -1 and "16-byte" in kmb.last_error()
    assert L.kmb_delta_backward(C.byref(p), None, 4096, None) == -1
    for missing in ("do_", "dq", "dk", "dv"):
        g = kmb.KMBDeltaGrads()
        for n in ("do_", "dq", "dk", "dv"):
            setattr(g, n, None if n == missing else 4096)
        assert L.kmb_delta_backward(C.byref(p), C.byref(g), 4096, None) == -1 and "required" in kmb.last_error()
    g.dv, g.ld_dq = 4096, 3
    assert L.kmb_delta_backward(C.byref(p), C.byref(g), 4096, None) == -1 and "stride" in kmb.last_error()
    for bad in (dict(h0=4096), dict(hT=4096), dict(cu_seqlens=4096, n_seq=1)):
        q = _delta(kmb, **bad)
        assert L.kmb_delta_step(C.byref(q), 4096, 4, None, None) == -1 and "NULL" in kmb.last_error()
    assert L.kmb_delta_step(C.byref(p), None, 4, None, None) == -1
    assert L.kmb_delta_step(C.byref(p), 4096, -1, None, None) == -1
    assert L.kmb_delta_step(C.byref(_delta(kmb, batch=0)), None, 0, None, None) == 0
    assert L.kmb_delta_forward(C.byref(_delta(kmb, batch=0)), None, 0, None) == 0


def test_norm_refusals(kmb):
    L = kmb.lib()

    def params(**kw):
        p = kmb.KMBNormParams()
        p.rows, p.D, p.dtype, p.eps, p.x, p.y = 4, 64, 0, 1e-5, 4096, 4096
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for bad in (dict(rows=-1), dict(D=0), dict(D=16385), dict(dtype=7), dict(eps=-1.0), dict(eps=math.nan),
                dict(mean=4096), dict(rstd=4096), dict(ld_x=63), dict(ld_y=1), dict(x=None), dict(y=None),
                dict(total=4096)):
        assert L.kmb_layernorm_forward(C.byref(params(**bad)), None) == -1, bad
        assert kmb.last_error().startswith("layernorm"), bad
    assert L.kmb_layernorm_forward(None, None) == -1
    assert L.kmb_layernorm_forward(C.byref(params(rows=0)), None) == 0
    g = kmb.KMBNormGrads()
    g.dy, g.dx = 4096, 4096
    ok = dict(mean=4096, rstd=4096)
    assert L.kmb_layernorm_backward(C.byref(params(**ok)), None, None, None) == -1
    assert L.kmb_layernorm_backward(C.byref(params()), C.byref(g), None, None) == -1          # no statistics
    assert L.kmb_layernorm_backward(C.byref(params(residual=4096, **ok)), C.byref(g), None, None) == -1   # no s
    g.ld_dx = 5
    assert L.kmb_layernorm_backward(C.byref(params(**ok)), C.byref(g), None, None) == -1
    g.ld_dx, g.dw = 0, 4096
    assert L.kmb_layernorm_backward(C.byref(params(**ok)), C.byref(g), None, None) == -1
    assert "workspace" in kmb.last_error()


def test_clip_refusals(kmb):
    L = kmb.lib()
    lst = (kmb.KMBGradTensor * 1)()
    call = lambda n=1, mx=1.0, ws=4096, l=lst: L.kmb_grad_clip(l, n, mx, 4096, ws, None)

    def entry(in_=4096, out=4096, n=8, dtype=0):
        lst[0].in_, lst[0].out, lst[0].n, lst[0].dtype = in_, out, n, dtype

    for bad in (dict(in_=None), dict(n=-1), dict(dtype=3), dict(in_=4098), dict(out=4097), dict(in_=4097, dtype=1)):
        entry(**bad)
        assert call() == -1 and kmb.last_error().startswith("kmb_grad_clip"), bad
    entry()
    for mx in (0.0, -1.0, math.nan):
        assert call(mx=mx) == -1
    assert call(n=-1) == -1 and call(ws=None) == -1 and call(ws=4100) == -1 and call(l=None) == -1
    assert L.kmb_model_clip_gradients(None, 1.0, None, None, None) == -1


def test_python_checks(kmb):
    t = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt)
    q, v = t(1, 4, 1, 8), t(1, 4, 1, 8)
    g = t(1, 4, 1)
    kmb.delta_params(q, q, v, g, g, v)
    with pytest.raises(ValueError):
        kmb.delta_params(q, t(1, 4, 1, 9), v, g, g, v)
    with pytest.raises(ValueError):
        kmb.delta_params(q, q, v, t(1, 4, 2), g, v)
    with pytest.raises(TypeError):
        kmb.delta_params(q.double(), q.double(), v.double(), g, g, v.double())
    with pytest.raises(ValueError):
        kmb.delta_params(q, q, v.to(torch.bfloat16), g, g, v)
    with pytest.raises(ValueError):
        kmb.delta_params(t(1, 4, 1, 16)[..., ::2], q, v, g, g, v)
    with pytest.raises(ValueError):
        kmb.delta_params(q, q, v, g, g, v, h0=t(2, 1, 8, 8))
    with pytest.raises(ValueError):
        kmb.norm_params(t(3, 8), t(9), None, t(3, 8))
    with pytest.raises(ValueError):
        kmb.norm_params(t(8, 3).t(), None, None, t(3, 8))
    with pytest.raises(ValueError):
        kmb.grad_list([t(4, 4).t()[:, :2]])


def test_plain_forms_against_differences():
    """The oracle's own gradients: autograd of the 64-bit definition against central differences of it."""
    gen = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)
    x = dict(q=n(1, 6, 1, 4), k=n(1, 6, 1, 4) * 0.5, v=n(1, 6, 2, 3), g=-n(1, 6, 2).abs(), beta=torch.sigmoid(n(1, 6, 2)),
             h0=n(2, 2, 4, 3))
    do, dh = n(1, 6, 2, 3), n(2, 2, 4, 3)

    def f(y):
        o, h = ref.delta(scale=0.7, cu=[0, 2, 6], **y)
        return (o * do).sum() + (h * dh).sum()

    for name in x:
        y = {k: t.clone() for k, t in x.items()}
        y[name].requires_grad_(True)
        g, = torch.autograd.grad(f(y), [y[name]])
        way, eps = n(*x[name].shape), 1e-6
        hi, lo = dict(x), dict(x)
        hi[name], lo[name] = x[name] + eps * way, x[name] - eps * way
        want = float(f(hi) - f(lo)) / (2 * eps)
        assert abs(float((g * way).sum()) - want) <= 1e-7 * float(g.norm() * way.norm())
