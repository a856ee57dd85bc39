"""Workloads of the gated delta mixer's operators: the gated delta rule (chunked forward and backward, and the recurrent
form over a pool of states), layer norm with its residual (forward and backward), and the global gradient norm with
clipping.

With ``own`` false, `run` is the plain form: elementary torch operations in 32 bits, rounded once at the end.  With
``own`` true it makes the calls a user makes of libkmamba_b200.so.  `exact` is the definition in 64 bits, token by token.
"""
import math
import random

import torch

own = False

DEV = "cuda"
CHUNK = 64


def _dt(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one request, one token, the mixer of a dim 512 layer: a decode step where latency is all
        {"name": "step_one", "op": "step", "dtype": "bf16", "B": 1, "T": 1, "Hk": 8, "Hv": 8, "dk": 64, "dv": 64},
        # a serving batch in full, some slots idle, value heads sharing key heads: state traffic
        {"name": "step_batch", "op": "step", "dtype": "bf16", "B": 250, "T": 1, "Hk": 8, "Hv": 16, "dk": 128, "dv": 128},
        # a short prompt of odd length going on from a state
        {"name": "prefill_short", "op": "prefill", "dtype": "bf16", "B": 1, "T": 777, "Hk": 8, "Hv": 8, "dk": 64,
         "dv": 64, "ragged": 0},
        # one long prompt: few heads, a long chain of chunks
        {"name": "prefill_long", "op": "prefill", "dtype": "bf16", "B": 1, "T": 16384, "Hk": 8, "Hv": 16, "dk": 128,
         "dv": 128, "ragged": 0},
        # a training step of the mixer over 64x64 grids, dim 512
        {"name": "train_dim512", "op": "train", "dtype": "bf16", "B": 8, "T": 4096, "Hk": 8, "Hv": 8, "dk": 64,
         "dv": 64, "ragged": 0},
        # training on packed sequences of uneven lengths, value heads sharing key heads
        {"name": "train_packed", "op": "train", "dtype": "bf16", "B": 1, "T": 8200, "Hk": 4, "Hv": 8, "dk": 128,
         "dv": 128, "ragged": 9},
        # the same in fp32 storage, odd sizes
        {"name": "train_f32", "op": "train", "dtype": "f32", "B": 2, "T": 1000, "Hk": 8, "Hv": 8, "dk": 60, "dv": 44,
         "ragged": 0},
        # the norm in front of a decode step
        {"name": "norm_row", "op": "norm", "dtype": "f32", "rows": 1, "D": 512, "residual": True, "train": False},
        # the norm of a training step over 32 grids of 64x64, dim 512
        {"name": "norm_train", "op": "norm", "dtype": "bf16", "rows": 131072, "D": 512, "residual": True, "train": True},
        # odd sizes, fp32 storage, no residual
        {"name": "norm_odd_f32", "op": "norm", "dtype": "f32", "rows": 10007, "D": 1001, "residual": False,
         "train": True},
        # the gradients of a 12-layer model of dim 512 in one arena, as many tensors; every step is clipped
        {"name": "clip_model", "op": "clip", "layers": 12, "dim": 512, "vocab": 256, "N": 64, "R": 4, "mixed": False,
         "clips": True},
        # a large model's gradients, half of them bf16, at odd sizes and places
        {"name": "clip_large", "op": "clip", "layers": 24, "dim": 2047, "vocab": 16384, "N": 64, "R": 16, "mixed": True,
         "clips": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "prefill", "train", "norm", "clip"])
    if op == "norm":
        D = _log(rng, 64, 4096)
        rows = max(1, min(_log(rng, 1, 131072), 131072 * 512 // D))
        return {"op": op, "dtype": rng.choice(["bf16", "f32"]), "rows": rows, "D": D,
                "residual": rng.random() < 0.5, "train": rng.random() < 0.7}
    if op == "clip":
        return {"op": op, "layers": rng.randint(1, 24), "dim": _log(rng, 64, 2047), "vocab": _log(rng, 64, 16384),
                "N": 64, "R": rng.choice([1, 2, 4]), "mixed": rng.random() < 0.5, "clips": rng.random() < 0.7}
    Hk = rng.choice([1, 2, 4, 8])
    Hv = Hk * rng.choice([1, 1, 2])
    if rng.random() < 0.6:
        dk = dv = rng.choice([64, 128])
    else:
        dk, dv = rng.randint(8, 128), rng.randint(8, 128)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "step":
        return {"op": op, "dtype": dtype, "B": _log(rng, 1, 250), "T": rng.choice([1, 1, 1, 2, 4, 5]), "Hk": Hk,
                "Hv": Hv, "dk": dk, "dv": dv}
    most = 16384 if op == "prefill" else 4096
    T = _log(rng, 32, most)
    B = rng.choice([1, 1, 2, 4])
    while B * T * Hv * dk * dv > (16384 * 16 * 128 * 128 if op == "prefill" else 8 * 4096 * 8 * 64 * 64):
        T = max(1, T // 2)
    ragged = rng.choice([0, 0, rng.randint(2, 12)]) if B == 1 else 0
    return {"op": op, "dtype": dtype, "B": B, "T": T, "Hk": Hk, "Hv": Hv, "dk": dk, "dv": dv, "ragged": ragged}


def work(case):
    op = case["op"]
    if op == "norm":
        n, e = case["rows"] * case["D"], 2 if case["dtype"] == "bf16" else 4
        fwd = n * e * (4 if case["residual"] else 2)
        bwd = n * e * (4 if case["residual"] else 3) - (0 if case["residual"] else n * e)
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": n * (8 + (12 if case["train"] else 0))}
    if op == "clip":
        plan = _tensor_plan(case)
        b = sum(n * (2 if bf else 4) for n, bf in plan)
        return {"bytes": b * (2 if case["clips"] else 1), "flops": 3 * sum(n for n, _ in plan)}
    e = 2 if case["dtype"] == "bf16" else 4
    n, Hk, Hv, dk, dv = case["B"] * case["T"], case["Hk"], case["Hv"], case["dk"], case["dv"]
    q = n * Hk * dk * e
    v = n * Hv * dv * e
    gate = 2 * n * Hv * 4
    seqs = case["ragged"] if case.get("ragged") else case["B"]
    state = seqs * Hv * dk * dv * 4
    if op == "train":   # q, k, v, gates, do in; o, dq, dk, dv, dgates out
        return {"bytes": 4 * q + 4 * v + 2 * gate, "flops": 18 * n * Hv * dk * dv}
    return {"bytes": 2 * q + 2 * v + gate + 2 * state, "flops": 6 * n * Hv * dk * dv}


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _lengths(case, seed):
    """Lengths of the packed sequences: uneven, an empty one and one of a single token among them."""
    n, T = case["ragged"], case["T"]
    r = random.Random(seed * 7 + n)
    cuts = sorted(r.randint(0, T) for _ in range(n - 1))
    cu = [0] + cuts + [T]
    if n >= 4:
        cu[2] = cu[1]
        cu[3] = max(cu[3], min(T, cu[2] + 1))
        cu = [cu[0]] + sorted(cu[1:])
    return cu


def _delta_inputs(case, seed):
    """Unit keys and queries, decays of the selective scan's own kind (a step size softplus(N(-4, 0.5)) times a rate in
    [1, 16]), write strengths sigmoid(N(0, 1))."""
    gen, dt = _gen(seed), _dt(case)
    B, T, Hk, Hv, dk, dv = (case[x] for x in ("B", "T", "Hk", "Hv", "dk", "dv"))

    def rand(*s):
        return torch.randn(s, generator=gen, device=DEV)

    def unit(x):
        return (x / x.square().sum(-1, keepdim=True).sqrt()).to(dt)

    rate = torch.exp(torch.rand((Hv,), generator=gen, device=DEV) * math.log(16.0))
    return {"q": unit(rand(B, T, Hk, dk)), "k": unit(rand(B, T, Hk, dk)), "v": rand(B, T, Hv, dv).to(dt),
            "g": -rate * torch.nn.functional.softplus(0.5 * rand(B, T, Hv) - 4.0),
            "beta": torch.sigmoid(rand(B, T, Hv)), "scale": dk ** -0.5, "rand": rand}


def _tensor_plan(case):
    """(elements, is bf16) of each gradient: an embedding, a head, then each layer's ten tensors."""
    V, D, N, R = case["vocab"], case["dim"], case["N"], case["R"]
    layer = [R * D, D * R, N, N * R * D, N * R * D, D, D, N * R, N * R, N // 2]
    sizes = [V * D, D * V] + layer * case["layers"]
    return [(n, case["mixed"] and i % 2 == 1) for i, n in enumerate(sizes)]


def prepare(case, seed):
    op = case["op"]
    st = {"case": case, "op": op}
    if op == "norm":
        gen, dt = _gen(seed), _dt(case)
        rows, D = case["rows"], case["D"]

        def rand(*s):
            return torch.randn(s, generator=gen, device=DEV)

        st.update(x=(rand(rows, D) * 2 + 0.5).to(dt), r=rand(rows, D).to(dt) if case["residual"] else None,
                  w=1 + 0.1 * rand(D), b=0.1 * rand(D), eps=1e-5)
        if case["train"]:
            st.update(dy=rand(rows, D).to(dt), ds=rand(rows, D).to(dt) if case["residual"] else None)
        return st
    if op == "clip":
        gen = _gen(seed)
        plan = _tensor_plan(case)
        at, places = {False: 1 if case["mixed"] else 0, True: 1}, []
        for n, bf in plan:   # each tensor at its place in the arena of its type; odd places where the case mixes types
            places.append((bf, at[bf], n))
            at[bf] += n if case["mixed"] else -(-n // 32) * 32
        arena = {bf: (torch.randn((at[bf],), generator=gen, device=DEV) * 0.01).to(torch.bfloat16 if bf else torch.float32)
                 for bf in (False, True)}
        out = {bf: torch.zeros_like(a) for bf, a in arena.items()}
        st.update(grads=[arena[bf][p:p + n] for bf, p, n in places], outs=[out[bf][p:p + n] for bf, p, n in places],
                  arenas=out, norm=torch.zeros(2, device=DEV))
        total = sum(n for _, _, n in places)
        st["max_norm"] = 0.01 * math.sqrt(total) * (0.3 if case["clips"] else 4.0)
        return st
    st.update(_delta_inputs(case, seed))
    rand = st.pop("rand")
    B, T, Hk, Hv, dk, dv = (case[x] for x in ("B", "T", "Hk", "Hv", "dk", "dv"))
    if op == "step":
        slots = random.Random(seed).sample(range(B + 6), B)
        slots = [-1 if i % 16 == 15 else s for i, s in enumerate(slots)]   # a request that has ended keeps its row
        st["slots"] = torch.tensor(slots, dtype=torch.int32, device=DEV)
        st["live"] = torch.tensor([i for i, s in enumerate(slots) if s >= 0], dtype=torch.int64, device=DEV)
        st["pool"] = 0.3 * rand(B + 6, Hv, dk, dv)
        return st
    seqs = B
    st["cu"] = None
    if case["ragged"]:
        cu = _lengths(case, seed)
        st["cu_host"], seqs = cu, case["ragged"]
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    st["h0"] = 0.3 * rand(seqs, Hv, dk, dv)
    if op == "train":
        st["do"] = rand(B, T, Hv, dv).to(_dt(case))
        st["dhT"] = 0.1 * rand(seqs, Hv, dk, dv)
    return st


# --------------------------------------------------------------------------- plain forms
def _rows(st, multiple):
    """Row of the token tensors for each place [sequence, position]; places past a sequence's end get the row that is
    appended behind the last (zeros).  And its inverse: the place of each token."""
    c = st["case"]
    B, T = c["B"], c["T"]
    if st.get("cu") is None:
        cu = [i * T for i in range(B + 1)]
    else:
        cu = st["cu_host"]
    longest = max(1, max(b - a for a, b in zip(cu, cu[1:])))
    Tp = -(-longest // multiple) * multiple
    start = torch.tensor(cu[:-1], device=DEV)[:, None]
    length = torch.tensor([b - a for a, b in zip(cu, cu[1:])], device=DEV)[:, None]
    pos = torch.arange(Tp, device=DEV)[None]
    idx = torch.where(pos < length, start + pos, B * T)
    back = torch.arange(B * T, device=DEV)
    seq = torch.searchsorted(torch.tensor(cu[1:], device=DEV), back, right=True)
    return idx, seq * Tp + back - torch.tensor(cu[:-1], device=DEV)[seq]


def _place(x, idx):
    flat = x.reshape((-1,) + x.shape[2:])
    return torch.cat([flat, torch.zeros_like(flat[:1])])[idx]


def _unit_lower_inverse(A):
    """(I + A)^-1 of strictly lower A, by doubling the size of the inverted diagonal blocks."""
    n = A.shape[-1]
    X = torch.eye(n, device=A.device, dtype=A.dtype).expand(A.shape)
    s = 1
    while s < n:
        blocks = A.reshape(A.shape[:-2] + (n // (2 * s), 2 * s, n // (2 * s), 2 * s))
        low = torch.diagonal(blocks, dim1=-4, dim2=-2).movedim(-1, -3)[..., s:, :s]
        inv = torch.diagonal(X.reshape(blocks.shape), dim1=-4, dim2=-2).movedim(-1, -3)
        a, b = inv[..., :s, :s], inv[..., s:, s:]
        top = torch.cat([a, torch.zeros_like(a)], -1)
        bottom = torch.cat([-(b @ (low @ a)), b], -1)
        full = torch.cat([top, bottom], -2)                      # [..., blocks, 2s, 2s]
        X = torch.diag_embed(full.movedim(-3, -1), dim1=-4, dim2=-2).reshape(A.shape)
        s *= 2
    return X


def _chunked(q, k, v, g, beta, h0, scale):
    """q, k [N, T, H, dk], v [N, T, H, dv], g, beta [N, T, H], T a multiple of CHUNK; h0 [N, H, dk, dv]."""
    def cut(x):
        x = x.reshape((x.shape[0], -1, CHUNK) + x.shape[2:])
        return x.movedim(3, 1)                                   # [N, H, chunks, C, ...]

    q, k, v, g, beta = (cut(x) for x in (q, k, v, g, beta))
    gam = g.cumsum(-1)
    low = torch.ones((CHUNK, CHUNK), dtype=torch.bool, device=DEV).tril()
    G = torch.exp((gam[..., :, None] - gam[..., None, :]).masked_fill(~low, -math.inf))
    kt = k.transpose(-1, -2)
    A = (beta[..., None] * G * (k @ kt)).masked_fill(~low.tril(-1), 0.0)
    X = _unit_lower_inverse(A)
    P = G * (q @ kt)
    eg = torch.exp(gam)[..., None]
    W, Ub = X @ (beta[..., None] * eg * k), X @ (beta[..., None] * v)
    qs, ks, last = q * eg, k * G[..., -1, :, None], eg[..., -1:, :]
    S, out = h0, []
    for i in range(q.shape[2]):                                  # the recurrence over chunks
        U = Ub[:, :, i] - W[:, :, i] @ S
        out.append(scale * (qs[:, :, i] @ S + P[:, :, i] @ U))
        S = last[:, :, i] * S + ks[:, :, i].transpose(-1, -2) @ U
    return torch.stack(out, 2).movedim(1, 3).flatten(1, 2), S    # [N, T, H, dv]


def _plain_delta(st):
    c, train = st["case"], st["op"] == "train"
    dt, grp = _dt(c), c["Hv"] // c["Hk"]
    idx, back = _rows(st, CHUNK)
    leaf = [st[x].float().requires_grad_(train) for x in ("q", "k", "v", "g", "beta", "h0")]
    if train:
        leaf = [x.detach().requires_grad_(True) for x in leaf]
    q, k, v, g, beta, h0 = leaf
    with torch.set_grad_enabled(train):
        qs, ks = (_place(x, idx).repeat_interleave(grp, 2) for x in (q, k))
        o, hT = _chunked(qs, ks, _place(v, idx), _place(g, idx), _place(beta, idx), h0, st["scale"])
        o = o.flatten(0, 1)[back].reshape(v.shape)
    if not train:
        return {"o": o.to(dt), "hT": hT}
    got = torch.autograd.grad([o, hT], leaf, [st["do"].float(), st["dhT"]])
    res = {"o": o.detach().to(dt), "hT": hT.detach()}
    res.update((n, x.to(dt)) for n, x in zip(("dq", "dk", "dv"), got))
    res.update(zip(("dg", "dbeta", "dh0"), got[3:]))
    return res


def _plain_step(st):
    c = st["case"]
    grp, live = c["Hv"] // c["Hk"], st["live"]
    q, k = (st[x][live].float().repeat_interleave(grp, 2) for x in ("q", "k"))
    v, g, beta = (st[x][live].float() for x in ("v", "g", "beta"))
    at = st["slots"][live].long()
    S, out = st["pool"][at], []
    for t in range(c["T"]):
        S = torch.exp(g[:, t])[..., None, None] * S
        u = beta[:, t][..., None] * (v[:, t] - (k[:, t][..., None] * S).sum(-2))
        S = S + k[:, t][..., None] * u[..., None, :]
        out.append(st["scale"] * (q[:, t][..., None] * S).sum(-2))
    st["pool"][at] = S
    o = torch.zeros_like(st["v"])
    o[live] = torch.stack(out, 1).to(o.dtype)
    return {"o": o, "pool": st["pool"]}


def _plain_norm(st):
    c, dt = st["case"], _dt(st["case"])
    x = st["x"].float()
    s = (x + st["r"].float()).to(dt) if c["residual"] else None
    x = s.float() if c["residual"] else x
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + st["eps"])
    xh = (x - mean) * rstd
    res = {"y": (xh * st["w"] + st["b"]).to(dt)}
    if c["residual"]:
        res["s"] = s
    if c["train"]:
        dy = st["dy"].float()
        wdy = dy * st["w"]
        dx = rstd * (wdy - wdy.mean(-1, keepdim=True) - xh * (wdy * xh).mean(-1, keepdim=True))
        if c["residual"]:
            dx = dx + st["ds"].float()
        res.update(dx=dx.to(dt), dw=(dy * xh).sum(0), db=dy.sum(0))
    return res


def _plain_clip(st):
    sq = torch.stack([g.float().square().sum() for g in st["grads"]]).sum()
    norm = sq.sqrt()
    coef = torch.where(norm > st["max_norm"], st["max_norm"] / norm, torch.ones_like(norm))
    for g, o in zip(st["grads"], st["outs"]):
        o.copy_((g.float() * coef).to(o.dtype))
    return {"norm": norm, "f32": st["arenas"][False], "bf16": st["arenas"][True]}


# --------------------------------------------------------------------------- the framework's calls
def _own_delta_handle(st):
    import bissimamba_b200 as kmb
    c, train = st["case"], st["op"] == "train"
    o, hT = torch.empty_like(st["v"]), torch.empty_like(st["h0"])
    p = kmb.delta_params(st["q"], st["k"], st["v"], st["g"], st["beta"], o, scale=st["scale"], h0=st["h0"], hT=hT,
                         cu_seqlens=st["cu"])
    ws = torch.empty(kmb.delta_workspace_floats(p, train), device=DEV)
    res = {"o": o, "hT": hT}
    grads = None
    if train:
        res.update((n, torch.empty_like(st[x])) for n, x in
                   (("dq", "q"), ("dk", "k"), ("dv", "v"), ("dg", "g"), ("dbeta", "beta"), ("dh0", "h0")))
        grads = kmb.delta_grads(p, st["do"], dhT=st["dhT"], **{n: res[n] for n in
                                                               ("dq", "dk", "dv", "dg", "dbeta", "dh0")})
    return kmb, p, grads, ws, res


def _own_delta(st):
    if "handle" not in st:   # what a program keeps for a layer: output buffers, workspace, the parameter structs
        st["handle"] = _own_delta_handle(st)
    kmb, p, grads, ws, res = st["handle"]
    stream = torch.cuda.current_stream().cuda_stream
    kmb.delta_forward(p, ws, keep=grads is not None, stream=stream)
    if grads is not None:
        kmb.delta_backward(p, grads, ws, stream=stream)
    return res


def _own_step(st):
    if "handle" not in st:
        import bissimamba_b200 as kmb
        o = torch.empty_like(st["v"])
        p = kmb.delta_params(st["q"], st["k"], st["v"], st["g"], st["beta"], o, scale=st["scale"])
        st["handle"] = (kmb, p, {"o": o, "pool": st["pool"]})
    kmb, p, res = st["handle"]
    kmb.delta_step(p, st["pool"], slots=st["slots"], stream=torch.cuda.current_stream().cuda_stream)
    return res


def _own_norm(st):
    if "handle" not in st:
        import bissimamba_b200 as kmb
        c, x = st["case"], st["x"]
        res = {"y": torch.empty_like(x)}
        if c["residual"]:
            res["s"] = torch.empty_like(x)
        stats = torch.empty((2, c["rows"]), device=DEV) if c["train"] else None
        p = kmb.norm_params(x, st["w"], st["b"], res["y"], eps=st["eps"], residual=st["r"], total=res.get("s"),
                            stats=stats)
        grads = ws = None
        if c["train"]:
            res.update(dx=torch.empty_like(x), dw=torch.empty_like(st["w"]), db=torch.empty_like(st["b"]))
            grads = kmb.norm_grads(p, st["dy"], dx=res["dx"], dw=res["dw"], db=res["db"], dtotal=st["ds"])
            ws = torch.empty(kmb.norm_workspace_floats(p), device=DEV)
        st["handle"] = (kmb, p, grads, ws, res)
    kmb, p, grads, ws, res = st["handle"]
    stream = torch.cuda.current_stream().cuda_stream
    kmb.norm_forward(p, stream=stream)
    if grads is not None:
        kmb.norm_backward(p, grads, ws, stream=stream)
    return res


def _own_clip(st):
    if "handle" not in st:
        import bissimamba_b200 as kmb
        lst = kmb.grad_list(st["grads"], st["outs"])
        st["handle"] = (kmb, lst, torch.empty(kmb.grad_clip_workspace_floats(lst), device=DEV))
    kmb, lst, ws = st["handle"]
    kmb.grad_clip(lst, st["max_norm"], st["norm"], ws, stream=torch.cuda.current_stream().cuda_stream)
    return {"norm": st["norm"][0], "f32": st["arenas"][False], "bf16": st["arenas"][True]}


def run(state):
    op = state["op"]
    if own:
        call = {"step": _own_step, "norm": _own_norm, "clip": _own_clip}.get(op, _own_delta)
    else:
        call = {"step": _plain_step, "norm": _plain_norm, "clip": _plain_clip}.get(op, _plain_delta)
    return call(state)


# --------------------------------------------------------------------------- the definition in 64 bits
def _exact_delta(st):
    """Token by token: S' = e^g S; u = beta (v - S'^T k); S = S' + k u^T; o = scale S^T q, and its adjoint."""
    c, train = st["case"], st["op"] == "train"
    grp = c["Hv"] // c["Hk"]
    idx, back = _rows(st, 1)
    q, k, v, g, beta = (_place(st[x].double(), idx) for x in ("q", "k", "v", "g", "beta"))
    q, k = q.repeat_interleave(grp, 2), k.repeat_interleave(grp, 2)
    S, scale, T = st["h0"].double(), st["scale"], idx.shape[1]
    if train and T * S.numel() * 8 > 60e9:
        return None
    before, us, out = [], [], []
    for t in range(T):
        if train:
            before.append(S)
        Sd = torch.exp(g[:, t])[..., None, None] * S
        u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None, :] @ Sd)[..., 0, :])
        S = Sd + k[:, t, :, :, None] * u[..., None, :]
        out.append(scale * (q[:, t, :, None, :] @ S)[..., 0, :])
        if train:
            us.append(u)

    def tokens(steps):
        return torch.stack(steps, 1).flatten(0, 1)[back]

    res = {"o": tokens(out).reshape(st["v"].shape), "hT": S}
    if not train:
        return res
    do = _place(st["do"].double(), idx)
    dS, dqs, dks, dvs, dgs, dbs = st["dhT"].double(), [], [], [], [], []
    after = S
    for t in reversed(range(T)):
        qt, kt, dot, u, bt = q[:, t], k[:, t], do[:, t], us[t], beta[:, t, :, None]
        al = torch.exp(g[:, t])[..., None, None]
        Sd = al * before[t]
        dqs.append(scale * (after @ dot[..., None])[..., 0])
        dS = dS + scale * qt[..., None] * dot[..., None, :]
        du = (kt[..., None, :] @ dS)[..., 0, :]
        dr = bt * du
        dks.append((dS @ u[..., None])[..., 0] - (Sd @ dr[..., None])[..., 0])
        dvs.append(dr)
        dbs.append((du * (v[:, t] - (kt[..., None, :] @ Sd)[..., 0, :])).sum(-1))
        dS = dS - kt[..., None] * dr[..., None, :]
        dgs.append((dS * Sd).sum((-1, -2)))
        dS = al * dS
        after = before[t]
    dq, dk = (tokens(x[::-1]).reshape(c["B"], c["T"], c["Hk"], grp, c["dk"]).sum(3) for x in (dqs, dks))
    res.update(dq=dq, dk=dk, dv=tokens(dvs[::-1]).reshape(st["v"].shape), dg=tokens(dgs[::-1]).reshape(st["g"].shape),
               dbeta=tokens(dbs[::-1]).reshape(st["g"].shape), dh0=dS)
    return res


def _exact_step(st):
    c = st["case"]
    grp = c["Hv"] // c["Hk"]
    pool, o = st["pool"].double(), torch.zeros(st["v"].shape, dtype=torch.float64, device=DEV)
    q, k = (st[x].double().repeat_interleave(grp, 2) for x in ("q", "k"))
    v, g, beta = (st[x].double() for x in ("v", "g", "beta"))
    for b, slot in enumerate(st["slots"].tolist()):
        if slot < 0:
            continue
        for t in range(c["T"]):
            S = torch.exp(g[b, t])[:, None, None] * pool[slot]
            u = beta[b, t][:, None] * (v[b, t] - torch.einsum("hk,hkv->hv", k[b, t], S))
            pool[slot] = S + torch.einsum("hk,hv->hkv", k[b, t], u)
            o[b, t] = st["scale"] * torch.einsum("hk,hkv->hv", q[b, t], pool[slot])
    return {"o": o, "pool": pool}


def _exact_norm(st):
    c = st["case"]
    x = st["x"].double()
    res = {}
    if c["residual"]:
        res["s"] = x + st["r"].double()
        x = res["s"].to(_dt(c)).double()   # the residual stream is what is stored
    mean = x.mean(-1, keepdim=True)
    sd = torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + st["eps"])
    xh, w = (x - mean) / sd, st["w"].double()
    res["y"] = xh * w + st["b"].double()
    if c["train"]:
        dy = st["dy"].double()
        t = dy * w
        dx = (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True)) / sd
        res["dx"] = dx + st["ds"].double() if c["residual"] else dx
        res["dw"], res["db"] = (dy * xh).sum(0), dy.sum(0)
    return res


def _exact_clip(st):
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in st["grads"]))
    coef = st["max_norm"] / norm if norm > st["max_norm"] else 1.0
    out = {bf: torch.zeros_like(a, dtype=torch.float64) for bf, a in st["arenas"].items()}
    for g, o in zip(st["grads"], st["outs"]):
        p = o.storage_offset()
        out[g.dtype == torch.bfloat16][p:p + g.numel()] = g.double() * coef
    return {"norm": norm, "f32": out[False], "bf16": out[True]}


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    return {"step": _exact_step, "norm": _exact_norm, "clip": _exact_clip}.get(op, _exact_delta)(st)
