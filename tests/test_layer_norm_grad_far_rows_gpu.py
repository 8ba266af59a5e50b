"""layer_norm_grad of rows that lie far from zero and hardly vary, against the formula in 64 bits, through the forward's
statistics.

u = 2^-24; a sum over a row has at most K = 80 additions one after another. The mean as it is handed over is off by u |c|, which
is taken away with the rest of the sum of x - mean: h is off by eh = rstd ((K u)^2 |c| + K u mean|x - mean|) + |h| rel, rel =
3 K u / 2 + 4 u + K u (rstd K u c)^2 the error of rstd. From it as everywhere, g = d w:
  * dx: rstd (4 u |g| + (K + 4) u (mean|g| + |h| mean|g h|) + |h| mean(|g| eh) + |c1| eh) + |dx| rel, and its rounding;
  * sums over rows: at most 200 additions one after another: 200 u sum|d h| + sum |d| eh, 200 u sum |d|, and rounding."""
import pytest
import torch

import dsa_triton_ascend_amd as dsa

pytestmark = pytest.mark.gpu
U, K = 2.0 ** -24, 80
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("width", [3, 7, 100, 257, 513, 700, 1001, 2000, 4099, 10001, 16384])
@pytest.mark.parametrize("c", [1e4 + 1 / 3, -77.0])
@pytest.mark.parametrize("spread", [0, 1, 5, "mixed"])
def test_rows_far_from_zero(dtype, width, c, spread):
    g = torch.Generator().manual_seed(width)
    c = float(torch.tensor(c).to(dtype))
    rows, eps = 13, 1e-6
    step = abs(c) * torch.finfo(dtype).eps   # about a unit in c's last place
    x = c + step * torch.randint(0, 6 if spread == "mixed" else spread + 1, (rows, width), generator=g).double()
    if spread == "mixed":   # rows far from zero beside others
        x[::2] = torch.randn(x[::2].shape, generator=g).double()
    x = x.to(dtype).cuda()
    d = torch.randn(rows, width, generator=g).to(dtype).cuda()
    w = (1 + 0.2 * torch.randn(width, generator=g)).cuda()
    b = (0.3 * torch.randn(width, generator=g)).cuda()
    xd, dd = x.double(), d.double()
    mean = xd.mean(-1, keepdim=True)
    rstd = 1 / (((xd - mean) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    h = (xd - mean) * rstd
    q = dd * w.double()
    m = lambda v: v.abs().mean(-1, keepdim=True)
    c0, c1 = q.mean(-1, keepdim=True), (q * h).mean(-1, keepdim=True)
    dx = (q - c0 - h * c1) * rstd
    top = xd.abs().amax(-1, keepdim=True)
    rel = 1.5 * K * U + 4 * U + K * U * (rstd * K * U * top) ** 2
    # (rows that are not far from zero keep the mean's rounding: it is within that of the sums, K u mean|x|)
    near = torch.where(mean.abs() * rstd > 4 - 1e-3, 0.0, K * U * m(xd))
    eh = rstd * ((K * U) ** 2 * top + K * U * m(xd - mean) + near) + h.abs() * rel
    tol_dx = rstd * (4 * U * q.abs() + (K + 4) * U * (m(q) + h.abs() * m(q * h)) + h.abs() * m(q.abs() * eh) + c1.abs() * eh) + dx.abs() * rel
    want = dict(dx=(dx, tol_dx), dw=((dd * h).sum(0), 200 * U * (dd * h).abs().sum(0) + (dd.abs() * eh).sum(0)),
                db=(dd.sum(0), 200 * U * dd.abs().sum(0)))
    y, got_mean, got_rstd = dsa.layer_norm(x, w, b, eps, return_stats=True)
    for name, got in zip(("dx", "dw", "db"), dsa.layer_norm_grad(d, x, got_mean, got_rstd, w, b)):
        v, tol = want[name]
        fi = torch.finfo(got.dtype)
        tol = tol + (v.abs() + tol) * fi.eps / 2 + fi.smallest_normal * fi.eps
        over = float(((got.double() - v).abs() - tol).max())
        assert over <= 0, f"{name} over its bound by {over:.3e}"
