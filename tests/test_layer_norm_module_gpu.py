"""A training step with the LayerNorm module: the gradients set by hand, as autograd does not follow it."""
import pytest
import torch

import dsa_triton_ascend_amd as dsa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", [True, False])
def test_step(bias):
    m = dsa.LayerNorm(96, bias=bias, device="cuda")
    opt = torch.optim.SGD(m.parameters(), lr=0.5)
    x, d = torch.randn(40, 96, device="cuda"), torch.randn(40, 96, device="cuda")
    before = [p.detach().clone() for p in m.parameters()]
    y, mean, rstd = m(x, return_stats=True)
    opt.step()   # without gradients: nothing
    assert all(torch.equal(p, b) for p, b in zip(m.parameters(), before))
    dx, dw, db = dsa.layer_norm_grad(d, x, mean, rstd, m.weight.detach(), None if m.bias is None else m.bias.detach())
    m.weight.grad = dw
    if bias:
        m.bias.grad = db
    opt.step()
    after = list(m.parameters())
    assert torch.equal(after[0].detach(), before[0] - 0.5 * dw)
    assert not bias or torch.equal(after[1].detach(), before[1] - 0.5 * db)
