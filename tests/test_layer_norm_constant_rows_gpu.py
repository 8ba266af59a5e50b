"""layer_norm of rows that lie far from zero and hardly vary, against the formula in 64 bits.

u = 2^-24; a sum over a row has at most K = 80 additions one after another. The mean is first off by at most m = K u |c|;
what is left after taking it away is exact and has a mean of its own, taken away in turn, so the centered values are off by
(K u)^2 |c| + K u mean|x - mean|. y is off by rstd times that, by |h| (3 K u / 2 + 4 u + K u (rstd m)^2) of the variance
(the square of the first mean's error is taken from it), and by its roundings; mean by u |c| more."""
import pytest
import torch

import dsa_triton_ascend_amd as dsa

pytestmark = pytest.mark.gpu
U, K = 2.0 ** -24, 80
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("width", [1, 3, 7, 100, 257, 1001, 4099, 10001, 16384])
@pytest.mark.parametrize("c", [1e4 + 1 / 3, -3333.0, 0.1])
@pytest.mark.parametrize("spread", [0, 1, 5])
def test_rows_far_from_zero(dtype, width, c, spread):
    g = torch.Generator().manual_seed(width)
    c = float(torch.tensor(c).to(dtype))
    step = abs(c) * torch.finfo(dtype).eps   # about a unit in c's last place
    x = (c + step * torch.randint(0, spread + 1, (9, width), generator=g).double()).to(dtype).cuda()
    w = (1 + 0.2 * torch.randn(width, generator=g)).cuda()
    b = (0.3 * torch.randn(width, generator=g)).cuda()
    eps = 1e-6
    xd = x.double()
    mean = xd.mean(-1, keepdim=True)
    rstd = 1 / (((xd - mean) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    h = (xd - mean) * rstd
    want = h * w.double() + b.double()
    m = K * U * abs(c)
    off = rstd * ((K * U) ** 2 * abs(c) + K * U * (xd - mean).abs().mean(-1, keepdim=True))
    rel = 1.5 * K * U + 4 * U + K * U * (rstd * m) ** 2
    tol = w.double().abs() * (off + h.abs() * rel) + 2 * U * (want.abs() + (h * w).abs())
    fi = torch.finfo(dtype)
    tol = tol + (want.abs() + tol) * fi.eps / 2 + fi.smallest_normal * fi.eps
    y, got_mean, got_rstd = dsa.layer_norm(x, w, b, eps, return_stats=True)
    over = float(((y.double() - want).abs() - tol).max())
    assert over <= 0, f"over its bound by {over:.3e}"
    assert ((got_mean.double() - mean[:, 0]).abs() <= U * abs(c) * 2 + off[:, 0] / rstd[:, 0]).all()
    assert ((got_rstd.double() / rstd[:, 0] - 1).abs() <= rel[:, 0]).all()
    # what the mean's own rounding leaves of h in the gradient is the statistics' business: constant rows have none
    if spread == 0:
        dx, dw, db = dsa.layer_norm_grad(torch.ones_like(x), x, got_mean, got_rstd, w, b)
        assert (dw == 0).all()
