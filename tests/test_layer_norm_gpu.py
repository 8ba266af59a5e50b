"""layer_norm and layer_norm_grad against the formulas in 64 bits.

Tolerances, per element, u = 2^-24. A sum over a row has at most K = 80 additions one after another (64 in a thread, 6
between lanes, up to 16 between waves less the short ones):
  * mean: dm = K u mean|x|; centered values: dm + u |x - mean|; so h = (x - mean) rstd is off by
    eh = rstd dm + |h| (3 K u / 2 + (rstd dm)^2 + 4 u)   (half the variance's relative error, its own shift, the root)
  * y = h w + b: |w| eh + 2 u |y|, and its rounding, half a step;
  * dx = (g - c0 - h c1) rstd with c0, c1 means over the row: rstd (4 u |g| + (K + 4) u (mean|g| + |h| mean|g h|) +
    |h| mean(|g| eh) + |c1| eh) + |dx| (3 K u / 2 + (rstd dm)^2 + 4 u), and its rounding;
  * sums over rows: at most 200 additions one after another: 200 u sum|d h| + sum |d| eh, 200 u sum |d|, and rounding.
"""
import pytest
import torch

import dsa_triton_ascend_amd as dsa

pytestmark = pytest.mark.gpu
U, K = 2.0 ** -24, 80
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def exact(x, w, b, d, eps):
    x = x.double()
    n = x.shape[-1]
    one = torch.ones(n, dtype=torch.double, device=x.device)
    w = one if w is None else w.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / (((x - mean) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    y = h * w + (0 if b is None else b.double())
    dm = K * U * x.abs().mean(-1, keepdim=True)
    rel = 1.5 * K * U + (rstd * dm) ** 2 + 4 * U
    eh = rstd * dm + h.abs() * rel
    out = dict(y=(y, w.abs() * eh + 2 * U * y.abs()), mean=(mean[..., 0], dm[..., 0]),
               rstd=(rstd[..., 0], (rstd * rel)[..., 0]))
    if d is not None:
        d = d.double()
        g = d * w
        c0, c1 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
        dx = (g - c0 - h * c1) * rstd
        m = lambda v: v.abs().mean(-1, keepdim=True)
        out["dx"] = (dx, rstd * (4 * U * g.abs() + (K + 4) * U * (m(g) + h.abs() * m(g * h)) + h.abs() * m(g.abs() * eh) + c1.abs() * eh)
                     + dx.abs() * rel)
        flat = lambda v: v.reshape(-1, n)
        out["dw"] = (flat(d * h).sum(0), 200 * U * flat((d * h).abs()).sum(0) + flat(d.abs() * eh).sum(0))
        out["db"] = (flat(d).sum(0), 200 * U * flat(d.abs()).sum(0))
    return out


def close(got, want, name):
    v, tol = want
    fi = torch.finfo(got.dtype)
    tol = tol + (v.abs() + tol) * fi.eps / 2 + fi.smallest_normal * fi.eps
    over = ((got.double() - v).abs() - tol).max() if v.numel() else 0.0
    assert torch.isfinite(got).all() and over <= 0, f"{name} over its bound by {float(over):.3e}"


def make(shape, dtype, wdt, seed, offset=0.25, extra=0, shift=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    x = (r(*shape[:-1], shape[-1] + extra) * 1.5 + offset).to(dtype).cuda()
    d = r(*shape[:-1], shape[-1] + extra).to(dtype).cuda()
    x, d = x[..., shift:shift + shape[-1]], d[..., shift:shift + shape[-1]]
    w = None if wdt is None else (1 + 0.2 * r(shape[-1])).to(wdt).cuda()
    b = None if wdt is None else (0.3 * r(shape[-1])).to(wdt).cuda()
    return x, d, w, b


def run_and_check(x, d, w, b, eps=1e-6):
    want = exact(x, w, b, d, eps)
    y, mean, rstd = dsa.layer_norm(x, w, b, eps, return_stats=True)
    assert y.shape == x.shape and y.is_contiguous() and mean.shape == x.shape[:-1]
    assert torch.equal(dsa.layer_norm(x, w, b, eps), y)
    dx, dw, db = dsa.layer_norm_grad(d, x, mean, rstd, w, b)
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    for name, got in dict(y=y, mean=mean, rstd=rstd, dx=dx, dw=dw, db=db).items():
        if got is not None:
            close(got, want[name], name)
    return y, dx, dw, db


# every thread layout: whole waves and parts of one, several rows a work-group, rows of 256, 512 and 1024 threads
WIDTHS = [1, 2, 3, 7, 8, 16, 33, 64, 65, 128, 136, 250, 256, 257, 500, 512, 513, 1000, 1001, 1024, 1025, 2048, 2056, 4096, 4104, 5120,
          7168, 8192, 8200, 10001, 16376, 16384]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(dtype, width):
    rows = 1 + (width * 7) % 19
    x, d, w, b = make((rows, width), dtype, F32 if width % 2 else dtype, width)
    run_and_check(x, d, w, b)


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 15, 16, 17, 63, 255, 1023, 4099, 20011])
@pytest.mark.parametrize("width", [96, 128, 1536])
def test_row_counts(rows, width):
    run_and_check(*make((rows, width), BF, F32, rows))


@pytest.mark.parametrize("dtype,wdt", [(BF, None), (HF, BF), (F32, HF), (BF, HF)])
def test_weight_types_and_none(dtype, wdt):
    x, d, w, b = make((37, 264), dtype, wdt, 5)
    run_and_check(x, d, w, b)
    if w is not None:
        run_and_check(x, d, w, None)


@pytest.mark.parametrize("shape,extra,shift", [((3, 5, 2, 128), 64, 0), ((41, 128), 8, 8), ((41, 128), 7, 3), ((9, 1000), 1, 1),
                                               ((2, 3, 512), 64, 64), ((1, 256), 3, 3)])
def test_strided_rows(shape, extra, shift):
    run_and_check(*make(shape, BF, BF, 9, extra=extra, shift=shift))


def test_uneven_transposed_and_expanded():
    x, d, w, b = make((4, 6, 64), HF, F32, 3)
    run_and_check(x.transpose(0, 1), d.transpose(0, 1), w, b)             # leading strides that do not join
    run_and_check(x.permute(2, 0, 1), d.permute(2, 0, 1), w[:6].contiguous(), b[:6].contiguous())   # last dimension strided
    run_and_check(x, d[:, :1].expand(4, 6, 64), w, b)                     # a gradient that was broadcast
    run_and_check(x[:1, :1].expand(5, 7, 64), d[0, 0].expand(5, 7, 64), w, b)
    u = torch.empty(2 * 64, device="cuda")[::2]
    u.copy_(w)
    run_and_check(x, d, u, b)                                              # strided weights
    run_and_check(x, d, torch.cat([w[:1], w])[1:], b)                     # off the 16-byte border


def test_large_mean_and_constant_rows():
    x, d, w, b = make((50, 640), F32, F32, 8, offset=300.0)
    run_and_check(x, d, w, b)
    x = torch.full((3, 128), 2.5, device="cuda")
    y, dx, dw, db = run_and_check(x, d[:3, :128].contiguous(), w[:128].contiguous(), b[:128].contiguous(), eps=1e-3)
    assert torch.equal(y, b[:128].expand(3, 128)) and (dw == 0).all()


def test_empty_rows_and_other_values():
    w, b = torch.ones(96, device="cuda"), torch.zeros(96, device="cuda")
    x = torch.empty(0, 5, 96, dtype=BF, device="cuda")
    y, mean, rstd = dsa.layer_norm(x, w, b, return_stats=True)
    dx, dw, db = dsa.layer_norm_grad(x, x, mean, rstd, w, b)
    assert y.shape == dx.shape == x.shape and mean.shape == (0, 5) and (dw == 0).all() and (db == 0).all()
    x = torch.randn(6, 96, device="cuda").to(BF)
    clean = dsa.layer_norm(x, w, b)
    x[2, 5], x[4, 0] = float("nan"), float("inf")
    y = dsa.layer_norm(x, w, b)   # such rows, and no others
    assert y[[2, 4]].isnan().all() and torch.equal(y[[0, 1, 3, 5]], clean[[0, 1, 3, 5]])


def test_differences():
    """The directional derivative of sum(y d) along u, by differences of the operator's own 32-bit outputs at a step of
    2^-5: the third derivative of h along unit directions is bounded by 15 rstd^3 |u|^3-like terms; here rstd is about
    0.67 and the quotient is off by less than 1% of |grad| |u| (step^2 / 6 times 15), plus 2^-22 |y| |d| sqrt(n) / step."""
    x, d, w, b = make((5, 48), F32, F32, 21)
    y, mean, rstd = dsa.layer_norm(x, w, b, return_stats=True)
    dx, dw, db = dsa.layer_norm_grad(d, x, mean, rstd, w, b)
    g = torch.Generator().manual_seed(4)
    h = 2.0 ** -5
    f = lambda x, w, b: float((dsa.layer_norm(x, w, b).double() * d.double()).sum())
    for grad, args in ((dx, lambda s, u: (x + s * u, w, b)), (dw, lambda s, u: (x, w + s * u, b)), (db, lambda s, u: (x, w, b + s * u))):
        u = torch.randn(grad.shape, generator=g).cuda()
        u = u / u.norm()
        quotient = (f(*args(h, u)) - f(*args(-h, u))) / (2 * h)
        noise = 2.0 ** -22 * float((y.abs() * d.abs()).norm()) / h
        assert abs(quotient - float((grad * u).sum())) < 0.01 * float(grad.norm()) + noise


def test_same_result_each_time_and_on_another_stream():
    x, d, w, b = make((3001, 392), BF, F32, 2)
    y, mean, rstd = dsa.layer_norm(x, w, b, return_stats=True)
    first = dsa.layer_norm_grad(d, x, mean, rstd, w, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = dsa.layer_norm_grad(d, x, mean, rstd, w, b)
        y2 = dsa.layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, y2) and all(torch.equal(a, c) for a, c in zip(first, again))


def test_captured_and_replayed():
    x, d, w, b = make((700, 256), BF, F32, 6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):   # warm
        y, mean, rstd = dsa.layer_norm(x, w, b, return_stats=True)
        dsa.layer_norm_grad(d, x, mean, rstd, w, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = dsa.layer_norm(x, w, b, return_stats=True)
        out = (y,) + dsa.layer_norm_grad(d, x, mean, rstd, w, b)
    for seed in (1, 2, 3):
        x2, d2, _, _ = make((700, 256), BF, F32, seed)
        x.copy_(x2)
        d.copy_(d2)
        graph.replay()
        torch.cuda.synchronize()
        e, m, r = dsa.layer_norm(x2, w, b, return_stats=True)
        want = (e,) + dsa.layer_norm_grad(d2, x2, m, r, w, b)
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_module():
    x, _, _, _ = make((3, 4, 64), BF, F32, 12)
    m = dsa.LayerNorm(64, norm_eps=1e-5, device="cuda")
    with torch.no_grad():
        m.weight.normal_()
        m.bias.normal_()
    assert torch.equal(m(x), dsa.layer_norm(x, m.weight.detach(), m.bias.detach(), 1e-5))
