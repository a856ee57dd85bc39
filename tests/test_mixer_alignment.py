"""The mixer operators' C entries refuse pointers off their elements' boundaries: the device cannot read there (no GPU is
needed)."""
import ctypes as C

import pytest


@pytest.mark.parametrize("dtype", [0, 1])
def test_delta(kmb, dtype):
    L = kmb.lib()
    wide, narrow = 4096 + (1 if dtype else 2), 4098

    def params(**kw):
        p = kmb.KMBDeltaParams()
        p.batch, p.T, p.Hk, p.Hv, p.dk, p.dv, p.dtype, p.scale = 1, 8, 1, 2, 16, 16, dtype, 1.0
        p.q = p.k = p.v = p.o = 4096
        for n, a in kw.items():
            setattr(p, n, a)
        return p

    def grads(**kw):
        g = kmb.KMBDeltaGrads()
        g.do_ = g.dq = g.dk = g.dv = 4096
        for n, a in kw.items():
            setattr(g, n, a)
        return g

    refused = lambda rc: rc == -1 and "not aligned" in kmb.last_error()
    for n, a in [(n, wide) for n in ("q", "k", "v", "o")] + [(n, narrow) for n in ("g", "beta", "h0", "hT")]:
        assert refused(L.kmb_delta_forward(C.byref(params(**{n: a})), 4096, 0, None)), n
        assert refused(L.kmb_delta_backward(C.byref(params(**{n: a})), C.byref(grads()), 4096, None)), n
        if n[0] != "h":
            assert refused(L.kmb_delta_step(C.byref(params(**{n: a})), 4096, 4, None, None)), n
    assert refused(L.kmb_delta_forward(C.byref(params(cu_seqlens=narrow, n_seq=1)), 4096, 0, None))
    for n, a in [(n, wide) for n in ("do_", "dq", "dk", "dv")] + [(n, narrow) for n in ("dhT", "dg", "dbeta", "dh0")]:
        assert refused(L.kmb_delta_backward(C.byref(params()), C.byref(grads(**{n: a})), 4096, None)), n
    assert refused(L.kmb_delta_step(C.byref(params()), narrow, 4, None, None))
    assert refused(L.kmb_delta_step(C.byref(params()), 4096, 4, narrow, None))


@pytest.mark.parametrize("dtype", [0, 1])
def test_norm_and_clip(kmb, dtype):
    L = kmb.lib()
    wide, narrow = 4096 + (1 if dtype else 2), 4098
    refused = lambda rc: rc == -1 and "not aligned" in kmb.last_error()

    def params(**kw):
        p = kmb.KMBNormParams()
        p.rows, p.D, p.dtype, p.eps, p.x, p.y, p.mean, p.rstd = 4, 64, dtype, 1e-5, 4096, 4096, 4096, 4096
        for n, a in kw.items():
            setattr(p, n, a)
        return p

    for n, a in [("x", wide), ("y", wide), ("residual", wide), ("w", narrow), ("b", narrow), ("mean", narrow),
                 ("rstd", narrow)]:
        assert refused(L.kmb_layernorm_forward(C.byref(params(**{n: a})), None)), n
    assert refused(L.kmb_layernorm_forward(C.byref(params(residual=4096, total=wide)), None))
    for n, a in [("dy", wide), ("dtotal", wide), ("dx", wide), ("dw", narrow), ("db", narrow)]:
        g = kmb.KMBNormGrads()
        g.dy = g.dx = g.dw = 4096
        setattr(g, n, a)
        assert refused(L.kmb_layernorm_backward(C.byref(params()), C.byref(g), 4096, None)), n
    g = kmb.KMBNormGrads()
    g.dy = g.dx = g.dw = 4096
    assert refused(L.kmb_layernorm_backward(C.byref(params()), C.byref(g), narrow, None))
    lst = (kmb.KMBGradTensor * 1)()
    lst[0].in_, lst[0].out, lst[0].n, lst[0].dtype = 4096, 4096, 8, dtype
    assert refused(L.kmb_grad_clip(lst, 1, 1.0, narrow, 4096, None))
