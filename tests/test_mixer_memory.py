"""The mixer operators' Python calls refuse tensors that the kernels would read or write as something else, before anything
reaches a device (no GPU is needed)."""
import pytest
import torch


def _step(kmb, B=3, Hk=1, Hv=2, dk=8, dv=4):
    t = lambda *s: torch.zeros(s)
    q, v = t(B, 1, Hk, dk), t(B, 1, Hv, dv)
    return kmb.delta_params(q, q, v, t(B, 1, Hv), t(B, 1, Hv), torch.zeros_like(v))


def test_pool_and_slots(kmb):
    p = _step(kmb)
    pool = torch.zeros(5, 2, 8, 4)
    for bad in (pool.bfloat16(), pool.transpose(2, 3), pool.transpose(2, 3).contiguous(), pool[:, :1], pool.view(5, 64),
                torch.zeros(5, 2, 8, 8)[..., :4], pool.double(), pool.int()):
        with pytest.raises(ValueError, match="pool"):
            kmb.delta_step(p, bad)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32)
    for bad in (slots.long(), slots[:2], torch.zeros(4, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2],
                slots.float(), slots.short()):
        with pytest.raises(ValueError, match="slots"):
            kmb.delta_step(p, pool, slots=bad)


def _wrong(floats):
    """Workspaces that do not hold so many fp32 entries in a row."""
    yield torch.zeros(floats - 1)
    yield torch.zeros(floats, dtype=torch.bfloat16)
    yield torch.zeros(2 * floats)[::2]


def test_workspaces(kmb):
    t = torch.zeros
    q, v, g = t(1, 70, 1, 8), t(1, 70, 2, 4), t(1, 70, 2)
    p = kmb.delta_params(q, q, v, g, g, t(1, 70, 2, 4))
    grads = kmb.delta_grads(p, v, q, q, v)
    for keep in (False, True):
        for ws in _wrong(kmb.delta_workspace_floats(p, keep)):
            with pytest.raises(ValueError, match="workspace"):
                kmb.delta_forward(p, ws, keep=keep)
    for ws in _wrong(kmb.delta_workspace_floats(p, True)):
        with pytest.raises(ValueError, match="workspace"):
            kmb.delta_backward(p, grads, ws)
    x = t(9, 16)
    n = kmb.norm_params(x, t(16), None, t(9, 16), stats=t(2, 9))
    for ws in _wrong(kmb.norm_workspace_floats(n)):
        with pytest.raises(ValueError, match="workspace"):
            kmb.norm_backward(n, kmb.norm_grads(n, x, dx=t(9, 16), dw=t(16)), ws)
    lst = kmb.grad_list([t(100)])
    for ws in _wrong(kmb.grad_clip_workspace_floats(lst)):
        with pytest.raises(ValueError, match="workspace"):
            kmb.grad_clip(lst, 1.0, t(2), ws)
    for result in _wrong(2):
        with pytest.raises(ValueError, match="result"):
            kmb.grad_clip(lst, 1.0, result, t(kmb.grad_clip_workspace_floats(lst)))


def test_host_tensors_and_other_devices(kmb):
    """A host pointer is no device pointer; "meta" stands for another device."""
    t = torch.zeros
    q, v, g = t(1, 4, 1, 8), t(1, 4, 2, 4), t(1, 4, 2)
    p = kmb.delta_params(q, q, v, g, g, t(1, 4, 2, 4))
    grads = kmb.delta_grads(p, v, q, q, v)
    ws = t(kmb.delta_workspace_floats(p, True))
    x = t(9, 16)
    n = kmb.norm_params(x, None, None, t(9, 16), stats=t(2, 9))
    lst, clip_ws = kmb.grad_list([x]), t(kmb.grad_clip_workspace_floats(kmb.grad_list([x])))
    for call in (lambda: kmb.delta_forward(p, ws), lambda: kmb.delta_backward(p, grads, ws),
                 lambda: kmb.delta_step(p, t(1, 2, 8, 4)), lambda: kmb.norm_forward(n),
                 lambda: kmb.norm_backward(n, kmb.norm_grads(n, x, dx=t(9, 16))),
                 lambda: kmb.grad_clip(lst, 1.0, t(2), clip_ws),
                 lambda: kmb.grad_clip(kmb.grad_list([]), 1.0, t(2), clip_ws)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    m = lambda s: s.to("meta")
    for call in (lambda: kmb.delta_params(q, m(q), v, g, g, v), lambda: kmb.delta_params(q, q, v, g, m(g), v),
                 lambda: kmb.delta_params(q, q, v, g, g, v, h0=m(t(1, 2, 8, 4))),
                 lambda: kmb.delta_params(q, q, v, g, g, v, h0=t(2, 2, 8, 4), cu_seqlens=m(t(3, dtype=torch.int32))),
                 lambda: kmb.delta_grads(p, m(v), q, q, v), lambda: kmb.norm_params(x, m(t(16)), None, x),
                 lambda: kmb.norm_grads(n, m(x)), lambda: kmb.grad_list([x, m(x)]), lambda: kmb.grad_list([x], [m(x)])):
        with pytest.raises(ValueError, match="expected on cpu"):
            call()


def test_a_list_without_its_outputs(kmb):
    a = [torch.zeros(3) for _ in range(3)]
    for outs in (a[:2], [], a + a):
        with pytest.raises(ValueError, match="3 gradients"):
            kmb.grad_list(a, outs)
