"""dense_attention_grad where sum_t P dP cancels against dP: keys and values with a common part, weights that lie on few
tokens, rows cut into ranges.

The gradients of queries and keys are products of dS = P (dP - delta). The kernels round dS to the io type once, and the
result. With the exact delta each rounding is off by at most half a step, independently, so the error's norm is that of
rounding the exact dS and the exact result once, in another draw of the same distribution: over some ten thousand
elements within a few per cent of it, and the 32-bit sums (2^-19 of the terms) are far below. Twice that norm is allowed.
The rounded output alone would put delta off by half a step of dO . O on every token alike, which adds up along what the
keys have in common: tens of times that norm."""
import math

import pytest
import torch

from tests.test_dense_attention_gpu import BF, HF, call
from tests.test_dense_attention_grad_gpu import gradients

pytestmark = pytest.mark.gpu


def make(dtype, n1, n2, d, dr, tokens, kv, seed, common, sharp):
    """Packed; every key and every value has the same vector of `common` times the random part's size in it"""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(query=r(sum(tokens), n1, d) * sharp, key=r(sum(kv), n2, d) + common * r(1, n2, d),
             value=r(sum(kv), n2, d) + common * r(1, n2, d), query_rope=None, key_rope=None)
    if dr:
        t.update(query_rope=r(sum(tokens), n1, dr) * sharp, key_rope=r(sum(kv), n2, dr) + common * r(1, n2, dr))
    t["d_out"] = r(sum(tokens), n1, d)
    return {k: None if v is None else v.to(dtype).cuda() for k, v in t.items()}


def exact(t, tokens, kv, scale, mode):
    """Gradients of queries and keys (with their rotary parts) in 64 bits, and the same from dS rounded once"""
    cat = lambda a, b: a if b is None else torch.cat([a, b], -1)
    io = t["query"].dtype
    q, k = cat(t["query"], t["query_rope"]).double(), cat(t["key"], t["key_rope"]).double()
    v, g = t["value"].double(), t["d_out"].double()
    n1, n2 = q.shape[1], k.shape[1]
    f = 1.0   # fp16: the bound of dS at 2^15
    if io == HF:
        f = 2.0 ** math.floor(14 - math.log2(float(g.norm(dim=-1).max() * v.norm(dim=-1).max())))
    dq, dk, rq, rk = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(q), torch.zeros_like(k)
    r0 = k0 = 0
    for nq, nk in zip(tokens, kv):
        rows, keys = slice(r0, r0 + nq), slice(k0, k0 + nk)
        r0, k0 = r0 + nq, k0 + nk
        seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        if mode == 3:
            seen = seen.tril(nk - nq)
        for h in range(n1):
            n = h // (n1 // n2)
            p = torch.softmax((q[rows, h] @ k[keys, n].t() * scale).masked_fill(~seen, -math.inf), -1)
            dp = g[rows, h] @ v[keys, n].t()
            w = p * (dp - (p * dp).sum(-1, keepdim=True))
            wr = (w * f).to(io).double() / f
            dq[rows, h], rq[rows, h] = scale * (w @ k[keys, n]), scale * (wr @ k[keys, n])
            dk[keys, n] += scale * (w.t() @ q[rows, h])
            rk[keys, n] += scale * (wr.t() @ q[rows, h])
    return dict(query=(dq, rq.to(io).double()), key=(dk, rk.to(io).double()))


CASES = [  # n1, n2, d, dr, tokens, kv, mode, common part, sharpness, splits
    (4, 2, 128, 0, [1500], [1500], 3, 1.0, 1.0, 1),
    (2, 2, 128, 64, [1100], [1400], 3, 1.0, 1.0, 1),
    (3, 1, 64, 0, [900, 700], [900, 700], 3, 1.0, 1.0, 1),
    (4, 2, 64, 0, [1500], [1500], 0, 2.0, 1.0, 1),
    (4, 2, 128, 0, [700], [700], 3, 0.0, 6.0, 1),           # weight on few tokens
    (2, 2, 128, 64, [700], [700], 3, 0.5, 5.0, 1),
    (4, 2, 128, 0, [300], [300], 3, 1.0, 1.0, 0),           # cut into ranges
    (4, 2, 128, 64, [280, 260], [300, 260], 3, 1.0, 1.0, 0),
    (4, 4, 128, 0, [700], [700], 3, 1.0, 1.0, 3),
    (6, 2, 64, 0, [700], [900], 3, 1.0, 3.0, 5),
    (8, 1, 128, 0, [1, 3], [2000, 1500], 3, 1.0, 1.0, 0),   # few rows over many tokens
    (2, 1, 128, 0, [200, 100], [200, 100], 3, 1.0, 1.0, 1),  # short rows
    (2, 1, 128, 64, [200, 100], [200, 100], 0, 1.0, 4.0, 2),
    (8, 8, 128, 0, [4100], [4100], 3, 1.0, 1.0, 0),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_as_near_as_one_rounding(case, dtype):
    n1, n2, d, dr, tokens, kv, mode, common, sharp, splits = CASES[case]
    scale = 1 / math.sqrt(d + dr)
    t = make(dtype, n1, n2, d, dr, tokens, kv, 900 + case, common, sharp)
    do = t.pop("d_out")
    got = gradients(t, do, call(t, tokens, kv, True, scale, mode), tokens, kv, True, scale, mode, splits=splits)
    want = exact({**t, "d_out": do}, tokens, kv, scale, mode)
    over = {}
    for name, main, rope in (("query", got[0], got[3]), ("key", got[1], got[4])):
        v, rounded = want[name]
        x = (main if rope is None else torch.cat([main, rope], -1)).double()
        over[name] = float((x - v).norm() / (rounded - v).norm())
    assert max(over.values()) <= 2, f"error over that of one rounding: {over}"
