"""Gated delta rule (include/kmamba_delta.h) against its definition in 64 bits, token by token, and the definition's
derivative (autograd in 64 bits, and central differences).

Bounds, 2-norm of the error over that of the result.  fp32 results: every product is exact to 2^-22 and sums are fp32,
a result passes about ten such products and sums in its chunk, and the rule contracts what it carries from chunk to
chunk: 64 units of 2^-24 = 4e-6; the gates' gradients are differences of such sums: 1e-5.  bf16 results: the final
rounding, at most 2^-9 of each entry, and 2^-11 for a product of single pieces: 3e-3."""
import math

import pytest
import torch

import mixer_ref as ref

pytestmark = pytest.mark.gpu

F32, GATE, BF16 = 4e-6, 1e-5, 3e-3


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-30)


def _inputs(B, T, Hk, Hv, dk, dv, dtype, seed, seqs=None, gates=True):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=gen)
    seqs = B if seqs is None else seqs
    x = {"q": _unit(n(B, T, Hk, dk)).to(dtype), "k": _unit(n(B, T, Hk, dk)).to(dtype), "v": n(B, T, Hv, dv).to(dtype),
         "g": -0.3 * torch.rand(B, T, Hv, generator=gen) if gates else None,
         "beta": torch.sigmoid(n(B, T, Hv)) if gates else None, "h0": 0.5 * n(seqs, Hv, dk, dv)}
    x["do"], x["dhT"] = n(B, T, Hv, dv).to(dtype), 0.3 * n(seqs, Hv, dk, dv)
    return x


def _run(kmb, dev, x, scale=0.5, cu=None, backward=True, stream=None):
    """The framework's forward and backward; every buffer it only writes starts as NaN."""
    d = {k: None if v is None else v.to(dev) for k, v in x.items()}
    nan = lambda t: torch.full_like(t, float("nan"))
    o = nan(d["v"])
    seqs = d["q"].shape[0] if cu is None else len(cu) - 1
    hT = torch.full((seqs, d["v"].shape[2], d["q"].shape[3], d["v"].shape[3]), float("nan"), device=dev)
    cud = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    p = kmb.delta_params(d["q"], d["k"], d["v"], d["g"], d["beta"], o, scale=scale, h0=d["h0"], hT=hT, cu_seqlens=cud)
    ws = torch.full((max(1, kmb.delta_workspace_floats(p, backward)),), float("nan"), device=dev)
    kmb.delta_forward(p, ws, keep=backward, stream=stream)
    res = {"o": o, "hT": hT}
    if backward:
        gate = torch.full(d["v"].shape[:3], float("nan"), device=dev)
        res.update(dq=nan(d["q"]), dk=nan(d["k"]), dv=nan(d["v"]), dg=gate, dbeta=gate.clone(), dh0=nan(hT))
        g = kmb.delta_grads(p, d["do"], dhT=d["dhT"], **{n: res[n] for n in ("dq", "dk", "dv", "dg", "dbeta", "dh0")})
        kmb.delta_backward(p, g, ws, stream=stream)
    torch.cuda.synchronize()
    assert kmb.lib().kmb_device_status(None) == 0
    return res


def _reference(x, scale=0.5, cu=None, backward=True):
    names = [n for n in ("q", "k", "v", "g", "beta", "h0") if x[n] is not None]
    leaf = {n: x[n].double().requires_grad_(backward) for n in names}
    full = {n: leaf.get(n) for n in ("q", "k", "v", "g", "beta", "h0")}
    o, hT = ref.delta(scale=scale, cu=cu, **full)
    res = {"o": o.detach(), "hT": hT.detach()}
    if backward:
        o = o + 0.0 * leaf["q"].sum()   # the graph reaches every output, also where no sequence holds a token
        got = torch.autograd.grad([o, hT], [leaf[n] for n in names], [x["do"].double(), x["dhT"].double()],
                                  allow_unused=True)
        res.update(("d" + n, torch.zeros_like(leaf[n]) if g is None else g) for n, g in zip(names, got))
    return res


def _compare(got, want, dtype):
    errs = {n: ref.rel(got[n], want[n]) for n in want if n in got}
    for n, e in errs.items():
        bound = GATE if n in ("dg", "dbeta") else BF16 if dtype == torch.bfloat16 and n in ("o", "dq", "dk", "dv") else F32
        assert e <= bound, (n, e, errs)


# (B, T, Hk, Hv, dk, dv): single tokens, chunk ends, odd and least widths, shared key heads
SHAPES = [(1, 1, 1, 1, 64, 64), (2, 2, 1, 1, 1, 1), (1, 63, 2, 2, 64, 64), (1, 64, 1, 2, 128, 128),
          (2, 65, 1, 3, 128, 16), (1, 130, 2, 2, 5, 3), (1, 200, 2, 4, 100, 37), (3, 129, 1, 1, 65, 128),
          (1, 192, 1, 1, 16, 65), (1, 77, 1, 1, 60, 44)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(kmb, cuda, shape, dtype):
    x = _inputs(*shape, dtype, seed=sum(shape))
    _compare(_run(kmb, cuda, x), _reference(x), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("absent", [("g",), ("beta",), ("h0",), ("g", "beta", "h0")])
def test_absent_inputs(kmb, cuda, absent, dtype):
    x = _inputs(1, 100, 1, 2, 64, 32, dtype, seed=3)
    for n in absent:
        x[n] = None
    if "beta" in absent:   # beta = 1 on unit keys is a projection: the chain of them needs no decay to stay bounded
        x["k"] = _unit(x["k"].float()).to(dtype)
    _compare(_run(kmb, cuda, x), _reference(x), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cu", [[0, 0, 1, 65, 65, 193, 200], [0, 200], [0, 1, 2, 3, 200], [3, 70, 190]])
def test_packed_sequences(kmb, cuda, cu, dtype):
    """Empty sequences, single tokens, tokens of no sequence (NaN there reaches nothing, and o stays as it was)."""
    x = _inputs(1, 200, 1, 2, 64, 48, dtype, seed=len(cu), seqs=len(cu) - 1)
    clean = {n: None if t is None else t.clone() for n, t in x.items()}
    out = [t for t in range(200) if not cu[0] <= t < cu[-1]]
    for n in ("q", "k", "v", "g", "beta", "do"):
        x[n][:, out] = float("nan")
        clean[n][:, out] = 0
    got, want = _run(kmb, cuda, x, cu=cu), _reference(clean, cu=cu)
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        assert torch.isnan(got[n][:, out].float()).all(), n
        got[n][:, out] = 0
    _compare(got, want, dtype)


@pytest.mark.parametrize("cu", [[0, 500, 100], [-5, 90, 60, 10 ** 9], [150, 20, 100]])
def test_offsets_outside_are_held_inside(kmb, cuda, cu):
    """Offsets that leave [0, T] or step back are taken as clamped and non-decreasing."""
    x = _inputs(1, 100, 1, 1, 32, 32, torch.float32, seed=1, seqs=len(cu) - 1)
    fixed, run = [], 0
    for c in cu:
        run = max(run, min(max(c, 0), 100))
        fixed.append(run)
    got, want = _run(kmb, cuda, x, cu=cu), _reference(x, cu=fixed)
    inside = slice(fixed[0], fixed[-1])
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        got[n], want[n] = got[n][:, inside], want[n][:, inside]
    _compare(got, want, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_resets_and_masked_tokens(kmb, cuda, dtype):
    """g = -inf forgets the state (also at a chunk's first and last token, and twice in a row), g = -1e30 the same;
    beta = 0 leaves it; a token with neither key nor value does nothing."""
    x = _inputs(1, 150, 1, 2, 64, 32, dtype, seed=8)
    x["g"][0, [0, 5, 6, 63, 64, 100], 0] = -math.inf
    x["g"][0, 30, 1] = -1e30
    x["beta"][0, [0, 10, 62, 63, 64, 65], 1] = 0.0
    x["k"][0, 20:40] = 0
    got, want = _run(kmb, cuda, x), _reference(x)
    assert torch.isfinite(got["dg"]).all()
    # the derivative with respect to g at -inf is 0 (autograd of exp gives 0 times the state)
    want["dg"] = torch.nan_to_num(want["dg"])
    _compare(got, want, dtype)


def test_everything_masked(kmb, cuda):
    """beta = 0 everywhere and no initial state: o and the states are exactly zero."""
    x = _inputs(1, 100, 1, 1, 64, 64, torch.float32, seed=2)
    x["beta"].zero_()
    x["h0"] = None
    got = _run(kmb, cuda, x)
    assert float(got["o"].abs().max()) == 0.0 and float(got["hT"].abs().max()) == 0.0
    want = _reference(x)
    for n in ("dq", "dk", "dv", "dbeta"):
        assert ref.rel(got[n], want[n]) <= GATE, n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["same_key", "few_keys", "large", "small", "uneven_rows"])
def test_hard_values(kmb, cuda, kind, dtype):
    """One key for all tokens (the triangular system at its fullest), and magnitudes far from 1: rows are scaled, so
    neither the values' size nor one row next to another matters."""
    x = _inputs(1, 140, 1, 1, 64, 48, dtype, seed=11)
    if kind == "same_key":
        x["k"][:] = x["k"][:, :1]
    elif kind == "few_keys":
        x["k"][:] = x["k"][:, [i % 3 for i in range(140)]]
    elif kind in ("large", "small"):
        f = 1e12 if kind == "large" else 1e-12
        for n in ("v", "h0"):
            x[n] = (x[n].float() * f).to(x[n].dtype)
    else:
        f = 10.0 ** (torch.arange(140) % 9 - 4).float()
        x["v"] = (x["v"].float() * f[None, :, None, None]).to(dtype)
        x["q"] = (x["q"].float() * f.flip(0)[None, :, None, None]).to(dtype)
    _compare(_run(kmb, cuda, x), _reference(x), dtype)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_that_are_not_finite(kmb, cuda, dtype, bad):
    """One at token 70, column 3 of v: the blocks of 16 tokens before it, the other 16-column units and the other head
    keep their bits, and in its unit nothing finite is wrong."""
    x = _inputs(1, 140, 2, 2, 64, 48, dtype, seed=13)
    clean = _run(kmb, cuda, x, backward=False)
    ref_o = _reference(x, backward=False)["o"]
    x["v"][0, 70, 0, 3] = bad
    got = _run(kmb, cuda, x, backward=False)
    assert torch.equal(got["o"][0, :64], clean["o"][0, :64])
    assert torch.equal(got["o"][0, :, 1], clean["o"][0, :, 1]) and torch.equal(got["hT"][0, 1], clean["hT"][0, 1])
    assert torch.equal(got["o"][0, :, 0, 16:], clean["o"][0, :, 0, 16:])
    rest, want = got["o"][0, 64:, 0, :16].double().cpu(), ref_o[0, 64:, 0, :16]
    fine = torch.isfinite(rest)
    assert not fine[7:, 3].any()   # behind the token its own column has no value
    fine[:, 3] = False
    assert (rest - want)[fine].abs().max() <= 1e-2 * want.abs().max() if fine.any() else True


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
def test_slices_of_one_projection(kmb, cuda, dtype, shift):
    """q, k, v as slices of one token row, at an aligned and an odd place; outputs and gradients of the same kind."""
    B, T, Hk, Hv, dk, dv = 2, 70, 2, 2, 32, 24
    x = _inputs(B, T, Hk, Hv, dk, dv, dtype, seed=21)
    W = 2 * Hk * dk + Hv * dv + 5 + shift

    def fused(like):
        row = torch.full((B, T, W), float("nan"), dtype=dtype, device=cuda)
        q = row[..., shift:shift + Hk * dk].view(B, T, Hk, dk)
        k = row[..., shift + Hk * dk:shift + 2 * Hk * dk].view(B, T, Hk, dk)
        v = row[..., shift + 2 * Hk * dk:shift + 2 * Hk * dk + Hv * dv].view(B, T, Hv, dv)
        if like:
            q.copy_(x["q"]), k.copy_(x["k"]), v.copy_(x["v"])
        return row, q, k, v

    _, q, k, v = fused(True)
    grow, dq, dk_, dv_ = fused(False)
    _, _, _, o = fused(False)
    _, _, _, do = fused(False)
    do.copy_(x["do"])
    h0, g, beta = x["h0"].to(cuda), x["g"].to(cuda), x["beta"].to(cuda)
    hT = h0.clone()   # the final states in place of the initial ones
    p = kmb.delta_params(q, k, v, g, beta, o, scale=0.5, h0=hT, hT=hT)
    ws = torch.empty(kmb.delta_workspace_floats(p, True), device=cuda)
    kmb.delta_forward(p, ws, keep=True)
    grads = kmb.delta_grads(p, do, dq, dk_, dv_, dhT=x["dhT"].to(cuda))
    kmb.delta_backward(p, grads, ws)
    torch.cuda.synchronize()
    want = _reference(x)
    _compare({"o": o, "hT": hT, "dq": dq, "dk": dk_, "dv": dv_}, want, dtype)
    assert torch.isnan(grow[..., -5:].float()).all(), "gradients written outside their slice"


def test_gradient_against_differences(kmb, cuda):
    """<gradient, direction> against the central difference of the definition in 64 bits along that direction."""
    x = _inputs(1, 70, 1, 2, 24, 16, torch.float32, seed=31)
    got = _run(kmb, cuda, x)
    gen = torch.Generator().manual_seed(5)

    def f(y):
        o, hT = ref.delta(scale=0.5, **{n: y[n] for n in ("q", "k", "v", "g", "beta", "h0")})
        return float((o * x["do"].double()).sum() + (hT * x["dhT"].double()).sum())

    for n in ("q", "k", "v", "g", "beta", "h0"):
        way = torch.randn(x[n].shape, generator=gen, dtype=torch.float64)
        eps = 1e-5   # the difference's own error: eps^2 from its third derivative, 1e-16 / eps from rounding
        hi, lo = dict(x), dict(x)
        hi[n], lo[n] = x[n].double() + eps * way, x[n].double() - eps * way
        want = (f(hi) - f(lo)) / (2 * eps)
        g = got["d" + n].double().cpu()
        assert abs(float((g * way).sum()) - want) <= 1e-5 * float(g.norm() * way.norm()), n


def test_same_bits_every_time_and_on_a_stream(kmb, cuda):
    x = _inputs(2, 150, 1, 2, 128, 64, torch.bfloat16, seed=41)
    a = _run(kmb, cuda, x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = _run(kmb, cuda, x, stream=s.cuda_stream)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_captured_in_a_graph(kmb, cuda):
    """No allocation, no synchronisation: forward, backward and step run from a graph."""
    x = {n: t.to(cuda) for n, t in _inputs(1, 100, 1, 1, 64, 64, torch.bfloat16, seed=51).items()}
    o, hT = torch.empty_like(x["v"]), torch.empty_like(x["h0"])
    p = kmb.delta_params(x["q"], x["k"], x["v"], x["g"], x["beta"], o, h0=x["h0"], hT=hT)
    ws = torch.empty(kmb.delta_workspace_floats(p, True), device=cuda)
    dq, dk, dv = (torch.empty_like(x[n]) for n in ("q", "k", "v"))
    g = kmb.delta_grads(p, x["do"], dq, dk, dv)

    def both(stream):
        kmb.delta_forward(p, ws, keep=True, stream=stream)
        kmb.delta_backward(p, g, ws, stream=stream)

    both(None)
    torch.cuda.synchronize()
    first = [t.clone() for t in (o, hT, dq, dk, dv)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(torch.cuda.current_stream().cuda_stream)
    for t in (o, hT, dq, dk, dv):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, (o, hT, dq, dk, dv)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 64, 64), (3, 1, 2, 4, 128, 128), (5, 4, 1, 2, 100, 37),
                                   (2, 3, 1, 1, 5, 3), (4, 1, 1, 3, 128, 16)])
def test_step(kmb, cuda, shape, dtype):
    """Recurrent form against the definition: slots in any order, idle rows (negative, past the pool)."""
    B, T, Hk, Hv, dk, dv = shape
    x = _inputs(*shape, dtype, seed=B + dv)
    gen = torch.Generator().manual_seed(7)
    pool = torch.randn(B + 3, Hv, dk, dv, generator=gen)
    slots = torch.randperm(B + 3, generator=gen)[:B].int()
    if B > 2:
        slots[1], slots[2] = -1, B + 3
    live = [b for b in range(B) if 0 <= slots[b] < B + 3]
    d = {n: x[n].to(cuda) for n in ("q", "k", "v", "g", "beta")}
    o = torch.full_like(d["v"], float("nan"))
    p = kmb.delta_params(d["q"], d["k"], d["v"], d["g"], d["beta"], o, scale=0.7)
    dev_pool = pool.to(cuda)
    kmb.delta_step(p, dev_pool, slots=slots.to(cuda))
    torch.cuda.synchronize()
    want, wo = pool.double(), torch.zeros(x["v"].shape, dtype=torch.float64)
    at = slots[live].long()
    wo[live], want[at] = ref.delta(x["q"][live], x["k"][live], x["v"][live], x["g"][live], x["beta"][live],
                                   pool[at], 0.7)
    assert ref.rel(dev_pool, want) <= F32
    assert ref.rel(o, wo) <= (BF16 if dtype == torch.bfloat16 else F32)
    rest = [i for i in range(B + 3) if i not in at.tolist()]
    assert torch.equal(dev_pool.cpu()[rest], pool[rest])


def test_step_at_the_end_of_a_large_pool(kmb, cuda):
    """A pool of more than 2^31 entries: the last slot's offset does not fit 32 bits."""
    n = 33000   # x 4 x 128 x 128 = 2.16e9 floats
    pool = torch.empty(n, 4, 128, 128, device=cuda)
    pool[-1].zero_()
    x = _inputs(1, 1, 4, 4, 128, 128, torch.float32, seed=61)
    d = {k: x[k].to(cuda) for k in ("q", "k", "v", "g", "beta")}
    o = torch.empty_like(d["v"])
    p = kmb.delta_params(d["q"], d["k"], d["v"], d["g"], d["beta"], o)
    kmb.delta_step(p, pool, slots=torch.tensor([n - 1], dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    wo, wS = ref.delta(x["q"], x["k"], x["v"], x["g"], x["beta"], None, 1.0)
    assert ref.rel(o, wo) <= F32 and ref.rel(pool[-1], wS[0]) <= F32


def test_steps_continue_a_prompt(kmb, cuda):
    """Chunked prefill, then tokens one by one, equals the whole sequence at once."""
    x = _inputs(2, 90, 1, 2, 64, 32, torch.float32, seed=71)
    whole = _run(kmb, cuda, x, backward=False)
    part = {n: (t[:, :80] if n not in ("h0", "dhT") else t) for n, t in x.items()}
    part = {n: t.contiguous() for n, t in part.items()}
    pre = _run(kmb, cuda, part, backward=False)
    pool, outs = pre["hT"], []
    for t in range(80, 90):
        d = {n: x[n][:, t:t + 1].contiguous().to(cuda) for n in ("q", "k", "v", "g", "beta")}
        o = torch.empty_like(d["v"])
        kmb.delta_step(kmb.delta_params(d["q"], d["k"], d["v"], d["g"], d["beta"], o, scale=0.5), pool)
        outs.append(o)
    assert ref.rel(torch.cat([pre["o"]] + outs, 1), whole["o"]) <= 2 * F32
    assert ref.rel(pool, whole["hT"]) <= 2 * F32


def test_nothing_to_do(kmb, cuda):
    """No tokens: the states pass through, and so do their gradients."""
    x = _inputs(2, 0, 1, 1, 16, 16, torch.float32, seed=1)
    got = _run(kmb, cuda, x)
    assert torch.equal(got["hT"].cpu(), x["h0"]) and torch.equal(got["dh0"].cpu(), x["dhT"])
    assert got["o"].numel() == 0
