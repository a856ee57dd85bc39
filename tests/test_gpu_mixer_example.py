"""The mixer's operators together: examples/gated_delta_mixer.py trains and serves."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_trains_and_serves(cuda, kmb, dtype):
    import gated_delta_mixer as ex
    m, losses, norms = ex.train(steps=60, dtype=dtype)
    assert all(torch.isfinite(torch.tensor(losses))) and all(torch.isfinite(torch.tensor(norms)))
    # 32 symbols: a model that knows nothing is at ln 32 = 3.47
    assert losses[0] > 3.0 and sum(losses[-5:]) / 5 < losses[0] - 0.5, losses
    # the same sums in another order (fp32), or the mixer's inputs and outputs rounded to bf16 on both sides
    assert ex.serve(m) <= (1e-4 if dtype == torch.float32 else 5e-2)


def test_gradients_of_the_whole_step(cuda, kmb):
    """One step's gradients against torch's autograd through the 64-bit definition."""
    import gated_delta_mixer as ex
    import mixer_ref as ref
    m = ex.Model()
    gen = torch.Generator().manual_seed(2)
    tokens, cu, counts = ex.batch(m.vocab, gen)
    logits, _ = m.forward(tokens, cu)
    loss = (torch.nn.functional.cross_entropy(logits[:-1], tokens[1:], reduction="none") * counts[:-1]).sum()
    got = torch.autograd.grad(loss, list(m.w.values()))

    w = {k: v.detach().double().cpu().requires_grad_(True) for k, v in m.w.items()}
    t, H, dk, dv = tokens.cpu(), m.H, m.dk, m.dv
    norm = lambda x, a, b: torch.nn.functional.layer_norm(x, (x.shape[-1],), a, b, 1e-5)
    x = w["embed"][t]
    row = norm(x, w["n1w"], w["n1b"]) @ w["proj"].t()
    q, k, v, a, b = row.split([H * dk, H * dk, H * dv, H, H], 1)
    unit = lambda z: torch.nn.functional.normalize(z.reshape(1, -1, H, dk), dim=-1)
    o, _ = ref.delta(unit(q), unit(k), v.reshape(1, -1, H, dv), -torch.nn.functional.softplus(a - 3.0)[None],
                     torch.sigmoid(b)[None], None, dk ** -0.5, cu.tolist())
    y = norm(o.reshape(len(t), -1) @ w["out"].t() + x, w["n2w"], w["n2b"]) @ w["head"].t()
    want_loss = (torch.nn.functional.cross_entropy(y[:-1], t[1:], reduction="none") * counts.cpu().double()[:-1]).sum()
    want = torch.autograd.grad(want_loss, list(w.values()))
    assert abs(float(loss) - float(want_loss)) <= 1e-5 * float(want_loss)
    for name, g, e in zip(m.w, got, want):
        assert ref.rel(g, e) <= 5e-5, name   # a dozen fp32 operators in a row, each within a few units of 2^-20
