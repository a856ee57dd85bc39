"""kmb_model_clip_gradients (include/kmamba_clip.h): which bound it takes."""
import ctypes as C
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_bound_that_is_no_number_is_refused(kmb, cuda):
    """max_norm <= 0 asks for the optimizer's clip_norm; NaN is neither and must not clip by it."""
    L = kmb.lib()
    cfg = kmb.model_config([8], 16, 16, 4, 1, 1)
    m = L.kmamba_create(C.byref(cfg))
    assert m, kmb.last_error()
    opt = kmb.MBOptimConfig()
    L.kmamba_optim_config_set_defaults(C.byref(opt))
    opt.clip_norm = 0.125
    assert L.kmamba_init(m, 1) == 0 and L.kmamba_enable_training(m, C.byref(opt), 1e-3, 0.0) == 0
    tok = torch.randint(0, 16, (1, 9), dtype=torch.int32, device=cuda)
    L.kmb_model_forward_backward(m, tok.data_ptr(), 1, None)
    n = C.c_size_t()
    arena = torch.as_tensor(kmb.DeviceArray(L.kmb_model_grad_arena(m, C.byref(n)), n.value), device=cuda)
    before = arena.clone()
    res, ws = torch.zeros(2, device=cuda), torch.zeros(L.kmb_grad_clip_workspace_floats(1), device=cuda)
    assert L.kmb_model_clip_gradients(m, math.nan, res.data_ptr(), ws.data_ptr(), None) == -1
    assert "max_norm" in kmb.last_error()
    torch.cuda.synchronize()
    assert torch.equal(arena, before)
    L.kmamba_free(m)
