"""Layer norm with its residual (include/kmamba_norm.h) against 64 bits.

Bounds (2-norm of the error over that of the result): fp32 results pass two sums over a row in fp32, whose error grows
slower than sqrt(D) units: 64 units of 2^-24 = 4e-6; bf16 results the final rounding, half a unit of 8 bits: at most
2^-8 of each entry.  dx is a difference of three terms that cancel (wholly so for two columns), so its error is
taken relative to them."""
import pytest
import torch

import mixer_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = 4e-6, 2.0 ** -8


def _case(rows, D, dtype, residual, seed, mean=0.5):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=gen)
    x = {"x": (n(rows, D) * 2 + mean).to(dtype), "r": n(rows, D).to(dtype) if residual else None,
         "w": 1 + 0.2 * n(D), "b": 0.3 * n(D), "dy": n(rows, D).to(dtype), "dt": n(rows, D).to(dtype) if residual else None}
    return x


def _run(kmb, dev, x, eps=1e-5, accumulate=None):
    d = {k: None if v is None else v.to(dev) for k, v in x.items()}
    rows, D = x["x"].shape
    y = torch.full_like(d["x"], float("nan"))
    s = None if d["r"] is None else torch.full_like(y, float("nan"))
    stats = torch.full((2, rows), float("nan"), device=dev)
    p = kmb.norm_params(d["x"], d["w"], d["b"], y, eps=eps, residual=d["r"], total=s, stats=stats)
    kmb.norm_forward(p)
    dx = torch.full_like(y, float("nan"))
    dw = torch.full((D,), float("nan"), device=dev) if accumulate is None else accumulate[0].to(dev)
    db = torch.full((D,), float("nan"), device=dev) if accumulate is None else accumulate[1].to(dev)
    ws = torch.full((max(1, kmb.norm_workspace_floats(p)),), float("nan"), device=dev)
    g = kmb.norm_grads(p, d["dy"], dx=dx, dw=dw, db=db, dtotal=d["dt"], accumulate=accumulate is not None)
    kmb.norm_backward(p, g, ws)
    torch.cuda.synchronize()
    return {"y": y, "s": s, "dx": dx, "dw": dw, "db": db}


def _check(got, x, eps=1e-5, base=None):
    s, y = ref.norm(x["x"], x["w"], x["b"], eps, x["r"])
    dx, dw, db = ref.norm_grads(s, x["w"], x["dy"], eps, x["dt"])
    if base is not None:
        dw, db = dw + base[0], db + base[1]
    t = BF16 if x["x"].dtype == torch.bfloat16 else F32
    assert ref.rel(got["y"], y) <= t
    d = s.double()
    rstd = 1.0 / torch.sqrt(((d - d.mean(-1, keepdim=True)) ** 2).mean(-1, keepdim=True) + eps)
    terms = float((rstd * x["dy"].double() * (1.0 if x["w"] is None else x["w"].double())).norm())
    assert float((got["dx"].cpu().double() - dx).norm()) <= F32 * terms + (t * float(dx.norm()) if t == BF16 else 0.0)
    assert ref.rel(got["dw"], dw) <= F32 and ref.rel(got["db"], db) <= F32
    if x["r"] is not None:
        assert torch.equal(got["s"].cpu(), s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,D", [(1, 512), (5, 2), (300, 7), (9, 64), (3000, 256), (33, 257), (2500, 512), (8, 1000),
                                    (40, 1001), (17, 1024), (700, 1025), (3, 1032), (20, 4099), (301, 8192), (2, 16384)])
def test_forward_and_gradients(kmb, cuda, rows, D, residual, dtype):
    x = _case(rows, D, dtype, residual, rows + D)
    _check(_run(kmb, cuda, x), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_column(kmb, cuda, dtype):
    """D = 1: y = b and nothing reaches x but what comes past the norm."""
    x = _case(6, 1, dtype, True, 3)
    got = _run(kmb, cuda, x)
    assert torch.equal(got["y"].cpu(), x["b"].to(dtype).expand(6, 1))
    assert torch.equal(got["dx"].cpu(), x["dt"])
    assert float(got["dw"].abs().max()) == 0.0


@pytest.mark.parametrize("D", [512, 1001, 3000])
def test_constant_rows_and_large_means(kmb, cuda, D):
    """A constant row has y = b exactly; a mean far above the spread costs no accuracy beyond the input's own."""
    x = _case(4, D, torch.float32, False, 5)
    x["x"][1] = 3.25
    got = _run(kmb, cuda, x)
    assert torch.equal(got["y"][1].cpu(), x["b"])
    x = _case(4, D, torch.float32, False, 5, mean=1024.0)
    got = _run(kmb, cuda, x)
    # entries are 1024 + O(1): the fp32 mean may be off by a few units of 1024 * 2^-24 = 6e-5, 3e-5 of the spread
    s, y = ref.norm(x["x"], x["w"], x["b"], 1e-5)
    assert ref.rel(got["y"], y) <= 2e-4


def test_no_weights(kmb, cuda):
    x = _case(50, 96, torch.float32, False, 6)
    x["w"] = x["b"] = None
    _check(_run(kmb, cuda, x), x)


@pytest.mark.parametrize("D", [512, 1100])
def test_accumulate(kmb, cuda, D):
    x = _case(64, D, torch.bfloat16, True, 7)
    base = [torch.randn(D) * 10, torch.randn(D) * 10]
    _check(_run(kmb, cuda, x, accumulate=[b.clone() for b in base]), x, base=base)


def test_rows_of_wider_tensors_and_in_place(kmb, cuda):
    """Strided rows at odd places, y over x, s over the residual, dx over dtotal: the same bits as apart."""
    for dtype in (torch.float32, torch.bfloat16):
        x = _case(37, 200, dtype, True, 8)
        apart = _run(kmb, cuda, x)

        def inside(t, off, pad):
            big = torch.zeros(37, 200 + pad, dtype=dtype, device=cuda)
            view = big[:, off:off + 200]
            view.copy_(t)
            return view

        for off, pad in ((0, 8), (1, 3)):
            a, r, dy, dt = inside(x["x"], off, pad), inside(x["r"], off, pad), inside(x["dy"], off, pad), inside(x["dt"], off, pad)
            w, b = x["w"].to(cuda), x["b"].to(cuda)
            stats = torch.empty(2, 37, device=cuda)
            p = kmb.norm_params(a, w, b, a, residual=r, total=r, stats=stats)
            kmb.norm_forward(p)
            dw, db = torch.empty(200, device=cuda), torch.empty(200, device=cuda)
            g = kmb.norm_grads(p, dy, dx=dt, dw=dw, db=db, dtotal=dt)
            kmb.norm_backward(p, g, torch.empty(kmb.norm_workspace_floats(p), device=cuda))
            torch.cuda.synchronize()
            s, y = ref.norm(x["x"], x["w"], x["b"], 1e-5, x["r"])
            assert torch.equal(r.cpu(), s)
            t = BF16 if dtype == torch.bfloat16 else F32
            assert ref.rel(a, y) <= t and ref.rel(dt, apart["dx"]) <= 2 * t
            assert ref.rel(dw, apart["dw"]) <= F32 and ref.rel(db, apart["db"]) <= F32


def test_gradient_against_differences(kmb, cuda):
    x = _case(5, 40, torch.float32, False, 9)
    got = _run(kmb, cuda, x)
    gen = torch.Generator().manual_seed(1)
    f = lambda a, w, b: float((ref.norm(a, w, b, 1e-5)[1] * x["dy"].double()).sum())
    for n, g in (("x", "dx"), ("w", "dw"), ("b", "db")):
        way, eps = torch.randn(x[n].shape, generator=gen, dtype=torch.float64), 1e-5
        a = {k: x[k].double() for k in ("x", "w", "b")}
        hi, lo = dict(a), dict(a)
        hi[n], lo[n] = a[n] + eps * way, a[n] - eps * way
        want = (f(**{"a": hi["x"], "w": hi["w"], "b": hi["b"]}) - f(**{"a": lo["x"], "w": lo["w"], "b": lo["b"]})) / (2 * eps)
        have = got[g].double().cpu()
        assert abs(float((have * way).sum()) - want) <= 1e-5 * float(have.norm() * way.norm())


def test_no_rows_same_bits_and_nan_rows(kmb, cuda):
    x = _case(0, 64, torch.float32, False, 1)
    got = _run(kmb, cuda, x)
    assert float(got["dw"].abs().max()) == 0.0 and float(got["db"].abs().max()) == 0.0
    x = _case(5000, 512, torch.bfloat16, True, 2)
    a, b = _run(kmb, cuda, x), _run(kmb, cuda, x)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    x["x"][7, 3] = float("nan")   # stays in its row
    c = _run(kmb, cuda, x)
    keep = [i for i in range(5000) if i != 7]
    assert torch.equal(c["y"][keep], a["y"][keep]) and torch.isnan(c["y"][7].float()).all()
