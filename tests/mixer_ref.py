"""Plain 64-bit forms of the mixer's operators on the CPU, for the tests: the gated delta rule token by token, layer
norm with its residual, the global gradient norm."""
import math

import torch


def delta(q, k, v, g=None, beta=None, h0=None, scale=1.0, cu=None):
    """Definition in 64 bits (differentiable).  q, k [B, T, Hk, dk], v [B, T, Hv, dv]; returns o and the final states.
    Tokens that no sequence holds have a zero o."""
    q, k, v = q.double(), k.double(), v.double()
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    q, k = (x.repeat_interleave(Hv // Hk, 2) for x in (q, k))
    g = torch.zeros(B, T, Hv, dtype=torch.float64) if g is None else g.double()
    beta = torch.ones(B, T, Hv, dtype=torch.float64) if beta is None else beta.double()
    rows = [(b, 0, T) for b in range(B)] if cu is None else [(0, a, e) for a, e in zip(cu, cu[1:])]
    out = [[torch.zeros(Hv, dv, dtype=torch.float64) for _ in range(T)] for _ in range(B)]
    final = []
    for n, (b, a, e) in enumerate(rows):
        S = torch.zeros(Hv, dk, dv, dtype=torch.float64) if h0 is None else h0[n].double()
        for t in range(a, e):
            alpha = torch.exp(g[b, t])[:, None, None]
            S = torch.where(alpha == 0, torch.zeros_like(S), alpha * S)
            u = beta[b, t][:, None] * (v[b, t] - torch.einsum("hk,hkv->hv", k[b, t], S))
            S = S + torch.einsum("hk,hv->hkv", k[b, t], u)
            out[b][t] = scale * torch.einsum("hk,hkv->hv", q[b, t], S)
        final.append(S)
    if T == 0:
        return torch.zeros(B, 0, Hv, dv, dtype=torch.float64), torch.stack(final)
    return torch.stack([torch.stack(r) for r in out]), torch.stack(final)


def norm(x, w, b, eps, residual=None):
    """s (rounded to x's type) and y in 64 bits."""
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = s.double()
    mean = d.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((d - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = (d - mean) * rstd
    y = y * w.double() if w is not None else y
    return s, y + b.double() if b is not None else y


def norm_grads(s, w, dy, eps, dtotal=None):
    s = s.double().requires_grad_(True)
    wd = torch.ones(s.shape[-1], dtype=torch.float64) if w is None else w.double()
    wd.requires_grad_(True)
    mean = s.mean(-1, keepdim=True)
    xh = (s - mean) / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + eps)
    dx, dw = torch.autograd.grad((xh * wd * dy.double()).sum(), [s, wd])
    if dtotal is not None:
        dx = dx + dtotal.double()
    return dx, dw, dy.double().sum(0)


def clip(grads, max_norm):
    n = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    return n, (max_norm / n if math.isfinite(n) and n > max_norm else 1.0)


def rel(got, ref):
    """2-norm of the difference over the 2-norm of the reference (0 / 0 = 0)."""
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    d, n = float((got - ref).norm()), float(ref.norm())
    return d / n if n else (math.inf if d else 0.0)
