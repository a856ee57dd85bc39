"""kmamba_forward's logits against the model's definition in 64 bits (the reference's own library is not needed)."""
import numpy as np
import pytest

from oracle import pyoracle as po
from test_gpu_model import SHAPES, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims,V,dim,N,R,nl", SHAPES)
def test_logits(kmb, cuda, dims, V, dim, N, R, nl):
    params = po.gen_model_params(V, dim, N, R, nl, seed=3)
    m = _model(kmb, dims, V, dim, N, R, nl, params)
    L = int(np.prod(dims))
    tok = np.random.default_rng(1).integers(0, V, L).astype(np.uint32)
    logits = np.zeros((L, V), np.float32)
    assert kmb.lib().kmamba_forward(m, tok.ctypes.data, logits.ctypes.data) == 0, kmb.last_error()
    kmb.lib().kmamba_free(m)
    want = np.asarray(po.model_logits64(dims, V, dim, N, R, nl, params, tok), np.float64).reshape(L, V)
    # the correctness bar of fp32 results, as a norm
    assert np.linalg.norm(logits - want) <= 1e-4 * np.linalg.norm(want)
