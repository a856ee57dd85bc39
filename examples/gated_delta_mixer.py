"""A small gated-delta language model on libkmamba_b200.so: trained on packed sequences, then served token by token.

One residual layer: layer norm -> one projection (queries, keys, values, gates) -> gated delta rule -> output
projection + residual -> layer norm -> head.  Norm, matrix products, mixer and gradient clipping are the library's;
torch holds the tensors, the elementwise gates, the loss and the optimizer.

    python examples/gated_delta_mixer.py [--steps 60] [--bf16]

The task: each symbol is followed by a fixed other one, nine times out of ten.
"""
import argparse
import ctypes as C
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import bissimamba_b200 as kmb  # noqa: E402


def _stream():
    return torch.cuda.current_stream().cuda_stream


def product(a, b, trans=0):
    """a [M, K] b [N, K]^T (trans 0) or a [K, M]^T b [K, N] (trans 1) at fp32 accuracy on the tensor cores."""
    a, b = a.contiguous(), b.contiguous()
    (M, K), N = (a.shape, b.shape[0]) if trans == 0 else ((a.shape[1], a.shape[0]), b.shape[1])
    d = torch.empty(M, N, device=a.device)
    kmb.check(kmb.lib().kmb_gemm_f32(-1, trans, M, N, K, a.data_ptr(), a.shape[1], b.data_ptr(), b.shape[1],
                                     d.data_ptr(), N, 0, _stream()), "kmb_gemm_f32")
    return d


class Linear(torch.autograd.Function):
    """y = x w^T"""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return product(x, w)

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        return product(dy, w.t()), product(dy, x, 1)


# A parameter struct holds its tensors, the outputs among them.  A context that kept one would keep itself alive through
# them, and the workspace with it, until Python's collector comes by: the backward makes its own.
class Norm(torch.autograd.Function):
    """(y, s): s = x + residual, y = its layer norm"""

    @staticmethod
    def forward(ctx, x, residual, w, b):
        y, s, ctx.stats = torch.empty_like(x), torch.empty_like(x), torch.empty(2, x.shape[0], device=x.device)
        kmb.norm_forward(kmb.norm_params(x, w, b, y, residual=residual, total=s, stats=ctx.stats), stream=_stream())
        ctx.save_for_backward(s, w)
        return y, s

    @staticmethod
    def backward(ctx, dy, ds):
        s, w = ctx.saved_tensors
        dy, ds = dy.contiguous(), ds.contiguous()
        dx, dw = torch.empty_like(dy), torch.empty(2, s.shape[1], device=dy.device)
        p = kmb.norm_params(s, w, None, dx, stats=ctx.stats)   # the backward reads the sum, not what it was made of
        g = kmb.norm_grads(p, dy, dx=dx, dw=dw[0], db=dw[1], dtotal=ds)
        kmb.norm_backward(p, g, torch.empty(kmb.norm_workspace_floats(p), device=dy.device), stream=_stream())
        return dx, dx, dw[0], dw[1]


class GatedDelta(torch.autograd.Function):
    """(o, final states) of packed sequences"""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, cu, scale):
        o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        hT = torch.empty(cu.numel() - 1, v.shape[2], k.shape[3], v.shape[3], device=v.device)
        g, beta = g.contiguous(), beta.contiguous()
        p = kmb.delta_params(q, k, v, g, beta, o, scale=scale, hT=hT, cu_seqlens=cu)
        ctx.ws, ctx.scale = torch.empty(kmb.delta_workspace_floats(p, True), device=v.device), scale
        kmb.delta_forward(p, ctx.ws, keep=True, stream=_stream())
        ctx.save_for_backward(q, k, v, g, beta, cu)
        ctx.mark_non_differentiable(hT)
        return o, hT

    @staticmethod
    def backward(ctx, do, _):
        q, k, v, g, beta, cu = ctx.saved_tensors
        dq, dk, dv, dg, db = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v, g, beta))
        p = kmb.delta_params(q, k, v, g, beta, dv, scale=ctx.scale, cu_seqlens=cu)   # o is not read
        grads = kmb.delta_grads(p, do.contiguous(), dq, dk, dv, dg=dg, dbeta=db)
        kmb.delta_backward(p, grads, ctx.ws, stream=_stream())
        return dq, dk, dv, dg, db, None, None


class Model:
    def __init__(self, vocab=32, dim=64, heads=2, dk=32, dv=32, dtype=torch.float32, seed=0, device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        r = lambda *s: (torch.randn(s, generator=gen) * s[-1] ** -0.5).to(device).requires_grad_(True)
        one = lambda n, v: torch.full((n,), v, device=device).requires_grad_(True)
        self.H, self.dk, self.dv, self.dtype, self.vocab = heads, dk, dv, dtype, vocab
        self.w = {"embed": r(vocab, dim), "proj": r(heads * (2 * dk + dv + 2), dim), "out": r(dim, heads * dv),
                  "head": r(vocab, dim), "n1w": one(dim, 1.0), "n1b": one(dim, 0.0), "n2w": one(dim, 1.0),
                  "n2b": one(dim, 0.0)}

    def mixer_inputs(self, y):
        """Queries, keys (unit), values and gates of the token rows y [n, dim]."""
        H, dk, dv = self.H, self.dk, self.dv
        row = Linear.apply(y, self.w["proj"])
        q, k, v, a, b = row.split([H * dk, H * dk, H * dv, H, H], 1)
        unit = lambda x: F.normalize(x.reshape(1, -1, H, dk), dim=-1).to(self.dtype)
        return (unit(q), unit(k), v.reshape(1, -1, H, dv).to(self.dtype), -F.softplus(a - 3.0).reshape(1, -1, H),
                torch.sigmoid(b).reshape(1, -1, H))

    def logits(self, o, x):
        mixed = Linear.apply(o.reshape(x.shape[0], -1).float(), self.w["out"])
        y, _ = Norm.apply(mixed, x, self.w["n2w"], self.w["n2b"])
        return Linear.apply(y, self.w["head"])

    def forward(self, tokens, cu):
        """Packed tokens [n] -> logits [n, vocab] and the final states."""
        x = self.w["embed"][tokens]
        y, x = Norm.apply(x, torch.zeros_like(x), self.w["n1w"], self.w["n1b"])
        o, states = GatedDelta.apply(*self.mixer_inputs(y), cu, self.dk ** -0.5)
        return self.logits(o, x), states

    @torch.no_grad()
    def step(self, tokens, pool, slots):
        """One new token of each request, its state in pool[slots[i]] -> logits."""
        x = self.w["embed"][tokens]
        y, x = Norm.apply(x, torch.zeros_like(x), self.w["n1w"], self.w["n1b"])
        q, k, v, g, beta = (t.transpose(0, 1).contiguous() for t in self.mixer_inputs(y))   # [requests, 1, ...]
        o = torch.empty_like(v)
        kmb.delta_step(kmb.delta_params(q, k, v, g, beta, o, scale=self.dk ** -0.5), pool, slots=slots,
                       stream=_stream())
        return self.logits(o, x)


def batch(vocab, gen, device="cuda"):
    """Packed sequences of uneven lengths: tokens, offsets, and which positions have a successor."""
    after = torch.randperm(vocab, generator=torch.Generator().manual_seed(9))
    tokens, cu, counts = [], [0], []
    for _ in range(16):
        n = int(torch.randint(12, 40, (1,), generator=gen))
        seq = torch.randint(0, vocab, (n,), generator=gen)
        follow = torch.rand(n, generator=gen) < 0.9
        for i in range(1, n):
            if follow[i]:
                seq[i] = after[seq[i - 1]]
        tokens.append(seq)
        counts += [torch.ones(n - 1), torch.zeros(1)]   # position i predicts token i + 1
        cu.append(cu[-1] + n)
    return (torch.cat(tokens).to(device), torch.tensor(cu, dtype=torch.int32, device=device),
            torch.cat(counts).to(device))


def train(steps=60, dtype=torch.float32, max_norm=1.0, lr=1e-2, log=None):
    """Returns the model, the losses and the gradient norms."""
    m = Model(dtype=dtype)
    names = list(m.w)
    opt = torch.optim.AdamW([m.w[n] for n in names], lr=lr)
    gen = torch.Generator().manual_seed(1)
    result, losses, norms = torch.zeros(2, device="cuda"), [], []
    for i in range(steps):
        tokens, cu, counts = batch(m.vocab, gen)
        logits, _ = m.forward(tokens, cu)
        loss = (F.cross_entropy(logits[:-1], tokens[1:], reduction="none") * counts[:-1]).sum() / counts.sum()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        lst = kmb.grad_list([m.w[n].grad.contiguous() for n in names])
        for n, g in zip(names, lst._keep[0]):
            m.w[n].grad = g
        kmb.grad_clip(lst, max_norm, result, torch.empty(kmb.grad_clip_workspace_floats(lst), device="cuda"),
                      stream=_stream())
        opt.step()
        losses.append(float(loss.detach()))
        norms.append(float(result[0]))
        if log and (i % 10 == 0 or i == steps - 1):
            log("step %3d  loss %.4f  gradient norm %.3f" % (i, losses[-1], norms[-1]))
    return m, losses, norms


def serve(m, prompt_lengths=(9, 14, 5), new=6, seed=3):
    """The same tokens through the chunked form at once, and as prompts continued token by token: the largest difference
    of the logits over the last tokens."""
    gen = torch.Generator().manual_seed(seed)
    seqs = [torch.randint(0, m.vocab, (n + new,), generator=gen).cuda() for n in prompt_lengths]
    offsets = lambda ls: torch.tensor([0] + list(torch.tensor(ls).cumsum(0)), dtype=torch.int32, device="cuda")
    with torch.no_grad():
        whole, _ = m.forward(torch.cat(seqs), offsets([len(s) for s in seqs]))
        _, states = m.forward(torch.cat([s[:-new] for s in seqs]), offsets(list(prompt_lengths)))
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    pool = torch.zeros((6,) + tuple(states.shape[1:]), device="cuda")
    pool[slots.long()] = states
    worst, at = 0.0, list(torch.tensor([len(s) for s in seqs]).cumsum(0))
    for t in range(new):
        got = m.step(torch.stack([s[len(s) - new + t] for s in seqs]), pool, slots)
        want = torch.stack([whole[int(e) - new + t] for e in at])
        worst = max(worst, float((got - want).abs().max()))
    return worst


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--bf16", action="store_true", help="bf16 queries, keys and values")
    a = ap.parse_args()
    m, _, _ = train(a.steps, torch.bfloat16 if a.bf16 else torch.float32, log=print)
    print("token by token against at once: logits differ by at most %.2g" % serve(m))


if __name__ == "__main__":
    main()
