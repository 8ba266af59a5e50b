"""An indexer's warm-up step as it runs: the key projection's rows through layer_norm and rotary_embedding, the model's
own dense_attention with the statistics that the dense loss takes, dense_loss_backward, and its d_key_index back
through rotary_embedding_grad and layer_norm_grad; beside it dense_attention_grad for the model.

The loss and d_key_index come from the oracle, given the rotated keys and statistics in 64 bits (of the same rounded
inputs); from there the way back is in 64 bits. Bounds: d_key_index is within 1e-2 of its norm (the dense loss's own
bound), then three roundings to the io type of half a step each, rho = 1e-2 + 3 eps / 2 in all. The way back of a row
is rstd P (w d) with a projection P, so d_x is off by at most rho max|w| max rstd |d| in norm; d_w sums d h and d_b sums
d, off by at most rho sum_r |d_r| times max|h| and 1."""
import numpy as np
import pytest
import torch

import dsa_triton_ascend_amd as dsa
from oracle import dense_loss_ref as oracle

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5
FREQ = 10000.0 ** (-torch.arange(32, dtype=torch.float32) / 32)


def make(dtype, B, S, n1, n2, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    return dict(x=r(B, S, 1, 128) * 1.5 + 0.25, w=(1 + 0.1 * torch.randn(128, generator=g)).cuda(),
                b=(0.1 * torch.randn(128, generator=g)).cuda(), qi=r(B, S, 32, 128), wi=r(B, S, 32).abs() / 8,
                q=r(B, S, n1, 128), k=r(B, S, n2, 128), v=r(B, S, n2, 128), qr=r(B, S, n1, 64), kr=r(B, S, n2, 64),
                d=r(B, S, n1, 128), pos=torch.arange(S).expand(B, S).contiguous().cuda(), freq=FREQ.cuda())


def step(t, act):
    h, mean, rstd = dsa.layer_norm(t["x"], t["w"], t["b"], return_stats=True)
    ki = dsa.rotary_embedding(h, t["pos"], t["freq"])
    qr, kr = (dsa.rotary_embedding(t[n], t["pos"], t["freq"]) for n in ("qr", "kr"))
    out, top, total = dsa.dense_attention(t["q"], t["k"], t["v"], SCALE, act, act, qr, kr, return_softmax_lse=True)
    imax, isum = dsa.dense_lightning_indexer_softmax_lse(t["qi"], ki, t["wi"], act, act)
    dqi, dki, dwi, loss = dsa.dense_loss_backward(t["q"], t["k"], t["qi"], ki, t["wi"], top, total, imax, isum, SCALE, qr, kr, act, act)
    dh = dsa.rotary_embedding_grad(dki, t["pos"], t["freq"])
    dx, dw, db = dsa.layer_norm_grad(dh, t["x"], mean, rstd, t["w"], t["b"])
    dq, dk, dv, dqr, dkr = dsa.dense_attention_grad(t["q"], t["k"], t["v"], t["d"], out, top, total, SCALE, qr, kr, act, act)
    dqr, dkr = (dsa.rotary_embedding_grad(x, t["pos"], t["freq"]) for x in (dqr, dkr))
    return dict(ki=ki, qr=qr, kr=kr, top=top, total=total, loss=loss, dki=dki, dx=dx, dw=dw, db=db, out=out, dq=dq, dk=dk, dv=dv,
                dqr=dqr, dkr=dkr, mean=mean, rstd=rstd, dqi=dqi, dwi=dwi)


def stats(t, r, act):
    """softmax_max and softmax_sum [B, N2, S, G] in 64 bits, zeros for rows that see nothing"""
    q, k = (torch.cat([t[a], r[b]], -1).cpu().double() for a, b in (("q", "qr"), ("k", "kr")))
    B, S, n1, _ = q.shape
    n2 = k.shape[2]
    k = k.repeat_interleave(n1 // n2, 2)
    top, total = torch.zeros(2, B, n2, S, n1 // n2, dtype=torch.float64).unbind(0)
    for b in range(B):
        n = act[b]
        if n == 0:
            continue
        s = q[b, :n].transpose(0, 1) @ k[b, :n].permute(1, 2, 0) * SCALE
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -torch.inf)
        m = s.amax(-1)
        rows = lambda x: x.view(n2, n1 // n2, n).transpose(1, 2)
        top[b, :, :n], total[b, :, :n] = rows(m), rows((s - m[..., None]).exp().sum(-1))
    return top, total


def turned_back(d, pos, freq):
    ang = pos.cpu().double()[..., None, None] * freq.cpu().double()
    c, s = ang.cos(), ang.sin()
    out = d.clone()
    a, b = d[..., 0:64:2], d[..., 1:64:2]
    out[..., 0:64:2], out[..., 1:64:2] = a * c + b * s, b * c - a * s
    return out


@pytest.mark.parametrize("dtype,S,n1,n2,act", [(torch.bfloat16, 70, 8, 2, [70, 33]), (torch.float16, 129, 6, 6, [1, 129]),
                                               (torch.bfloat16, 64, 12, 4, [0, 64])])
def test_step(dtype, S, n1, n2, act):
    t = make(dtype, len(act), S, n1, n2, S)
    r = step(t, act)
    f = lambda x: x.float().cpu().numpy()
    top, total = stats(t, r, act)
    seen = total > 0
    assert torch.allclose(r["top"].cpu().double()[seen], top[seen], rtol=0, atol=1e-4)
    assert torch.allclose(r["total"].cpu().double()[seen], total[seen], rtol=1e-4, atol=0)
    imax, isum = oracle.dense_softmax_lse(f(t["qi"]), f(r["ki"]), f(t["wi"]), act, act)
    _, dki, _, loss = oracle.dense_loss_backward(f(t["q"]), f(t["k"]), f(r["qr"]), f(r["kr"]), f(t["qi"]), f(r["ki"]), f(t["wi"]),
                                                 top.numpy(), total.numpy(), imax, isum, SCALE, act, act, io_dtype="fp32")
    assert abs(float(r["loss"]) - float(loss[0])) <= 1e-2 * abs(float(loss[0])) + 1e-3
    # the way back of the oracle's d_key_index
    x = t["x"].cpu().double()
    mean = x.mean(-1, keepdim=True)
    rstd = (x.var(-1, unbiased=False, keepdim=True) + 1e-6).rsqrt()
    h, w = (x - mean) * rstd, t["w"].cpu().double()
    d = turned_back(torch.from_numpy(np.asarray(dki, np.float64)), t["pos"], t["freq"])
    g = d * w
    dx = (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True)) * rstd
    rho = 1e-2 + 3 * torch.finfo(dtype).eps / 2
    off = lambda got, want: (got.cpu().double() - want).norm()
    assert off(r["dx"], dx) <= rho * w.abs().max() * rstd.max() * d.norm()
    rows = d.norm(dim=-1).sum()
    assert off(r["dw"], (d * h).sum((0, 1, 2))) <= rho * rows * h.abs().max()
    assert off(r["db"], d.sum((0, 1, 2))) <= rho * rows
    for b, n in enumerate(act):   # rows that are no tokens
        for name in ("out", "dq", "dk", "dv", "dqr", "dkr", "dx"):
            assert not r[name][b, n:].any(), name


def test_step_in_a_graph():
    """The same step captured with its one-shot calls and replayed on new inputs gives what eager runs give"""
    act = [100, 37]
    t = make(torch.bfloat16, 2, 100, 8, 2, 1)
    step(t, act)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(t, act)
    for seed in (2, 3, 4):
        new = make(torch.bfloat16, 2, 100, 8, 2, seed)
        want = step(new, act)
        for name in t:
            t[name].copy_(new[name])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in want:
            if name not in ("dki", "dx", "dw", "db", "dqi", "dwi", "loss"):
                assert torch.equal(kept[name], want[name]), name
            else:   # (the loss's sums may be in another order)
                a, b = kept[name].double(), want[name].double()
                assert (a - b).norm() <= 1e-2 * b.norm() + 1e-6, name
