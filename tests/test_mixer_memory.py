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
                torch.zeros(5, 2, 8, 8)[..., :4]):
        with pytest.raises(ValueError, match="pool"):
            kmb.delta_step(p, bad)
    with pytest.raises(TypeError):
        kmb.delta_step(p, pool.double())
    slots = torch.tensor([4, 0, 2], dtype=torch.int32)
    for bad in (slots.long(), slots[:2], torch.zeros(4, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2],
                slots.float(), slots.short()):
        with pytest.raises(ValueError, match="slots"):
            kmb.delta_step(p, pool, slots=bad)
