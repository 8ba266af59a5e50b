"""dense_attention_grad against the formula in 64 bits.

Tolerances, per element, u = 2^-24, e = eps / 2 of the io type. With the exact P, dP, delta:
  * score errors ds (as in the forward's test) move P by 2 ds relative; the statistics add as much; exp2 and log2 2^-20: rp =
    4 ds + 2^-19;
  * dP: a sum of D products, ep = D u sum|dO v|; delta: from the rounded output, ed = e sum|dO O| + D u sum|dO O| + the
    output's own error |dO| (forward tolerance);
  * dS is off by P (ep + ed) + |dS| rp + P |dP - delta| 2^-22, and rounded: e |dS|, in fp16 at least half a step of 2^-24 over
    its factor: |dO||v| max 2^-25 2^-13; P for dV: P rp and e P, in fp16 at least 2^-25 2^-15;
  * each product's 32-bit sum of n terms: n u times the sum of magnitudes (n u of them at most; 2^-14 here covers n <= 1000
    in the worst order, longer sums by the square root of their length);
  * and the output's own rounding, e."""
import math

import pytest
import torch

import dsa_triton_ascend_amd as dsa
from tests.test_dense_attention_gpu import BF, HF, CASES, call, exact, make, strided

pytestmark = pytest.mark.gpu
NAMES = ("d_query", "d_key", "d_value", "d_query_rope", "d_key_rope")


def gradients(t, do, fwd, tokens, kv, packed, scale, mode=3, **kw):
    cu = (lambda n: torch.tensor(n).cumsum(0).tolist()) if packed else (lambda n: n)
    return dsa.dense_attention_grad(t["query"], t["key"], t["value"], do, *fwd, scale, t["query_rope"], t["key_rope"],
                                    cu(tokens), cu(kv), "TND" if packed else "BSND", mode, **kw)


def exact_grads(t, do, tokens, kv, packed, scale, mode=3):
    """{name: (value, tolerance)} in 64 bits, in the operands' shapes."""
    io = t["query"].dtype
    e, u = torch.finfo(io).eps / 2, 2.0 ** -24
    cat = lambda a, b: a if b is None else torch.cat([a, b], -1)
    q, k, v, g = cat(t["query"], t["query_rope"]).double(), cat(t["key"], t["key_rope"]).double(), t["value"].double(), do.double()
    S1, S2 = (0, 0) if packed else (q.shape[1], k.shape[1])
    q, k, v, g = (x if packed else x.flatten(0, 1) for x in (q, k, v, g))
    n1, n2, d, wide = q.shape[1], k.shape[1], v.shape[-1], q.shape[-1]
    out, _, _, otol, ds_f = exact(t, tokens, kv, packed, scale, mode)
    z = lambda x: torch.zeros_like(x)
    dq, dk, dv, tq, tk, tv = z(q), z(k), z(v), z(q), z(k), z(v)
    live_k = torch.zeros(k.shape[0], dtype=torch.bool, device="cuda")
    bound = 0.0
    if io == HF:
        bound = float(g.norm(dim=-1).max() * v.norm(dim=-1).max())
    aq = ak = 0
    per = n1 // n2
    for b, (nq, nk) in enumerate(zip(tokens, kv)):
        r0, k0 = (aq, ak) if packed else (b * S1, b * S2)
        aq, ak = aq + nq, ak + nk
        if not nq or not nk:
            continue
        rows, keys = slice(r0, r0 + nq), slice(k0, k0 + nk)
        seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        if mode == 3:
            seen = seen.tril(nk - nq)
        live = seen.any(-1)
        for h in range(n1):
            n = h // per
            qq, kk, vv, gg = q[rows, h], k[keys, n], v[keys, n], g[rows, h]
            s = (qq @ kk.t() * scale).masked_fill(~seen, -math.inf)
            m = s.amax(-1).masked_fill(~live, 0.0)
            p = torch.exp(s - m[:, None])
            p = p / p.sum(-1).masked_fill(~live, 1.0)[:, None]
            dp = gg @ vv.t()
            delta = (p * dp).sum(-1, keepdim=True)
            w = p * (dp - delta)
            rp = 4 * ds_f[rows, h][:, None] + 2.0 ** -19
            ep = d * u * (gg.abs() @ vv.abs().t())
            mag = (gg.abs() * out[rows, h].abs()).sum(-1, keepdim=True)
            ed = (e + d * u) * mag + (gg.abs() * otol[rows, h]).sum(-1, keepdim=True)
            ew = p * (ep + ed) + w.abs() * (rp + e) + p * (dp.abs() + delta.abs()) * 2.0 ** -22
            pe = p * (rp + e)
            if io == HF:
                ew = ew + seen * bound * 2.0 ** -38
                pe = pe + seen * 2.0 ** -40
            dv[keys, n] += p.t() @ gg
            tv[keys, n] += (pe + 2.0 ** -14 * p).t() @ gg.abs()
            dq[rows, h] = scale * (w @ kk)
            tq[rows, h] = abs(scale) * ((ew + 2.0 ** -14 * w.abs()) @ kk.abs())
            dk[keys, n] += scale * (w.t() @ qq)
            tk[keys, n] += abs(scale) * ((ew + 2.0 ** -14 * w.abs()).t() @ qq.abs())
    tiny = torch.finfo(io).smallest_normal * e
    res = {}
    for name, x, tol, like in (("d_query", dq[..., :d], tq[..., :d], "query"), ("d_key", dk[..., :d], tk[..., :d], "key"),
                               ("d_value", dv, tv, "value"), ("d_query_rope", dq[..., d:], tq[..., d:], "query_rope"),
                               ("d_key_rope", dk[..., d:], tk[..., d:], "key_rope")):
        if t[like] is not None:
            res[name] = (x.reshape(t[like].shape), (tol + e * (x.abs() + tol) + tiny).reshape(t[like].shape))
    return res


def check(got, want):
    for name, g in zip(NAMES, got):
        assert (g is None) == (name not in want)
        if g is None:
            continue
        v, tol = want[name]
        assert g.shape == v.shape and g.is_contiguous() and torch.isfinite(g).all(), name
        over = ((g.double() - v).abs() - tol).max()
        assert over <= 0, f"{name} over its bound by {float(over):.3e}"
        # the bounds are of the worst case: errors of the usual size add like a random walk
        if float(v.norm()) > 0:
            rel = float((g.double() - v).norm() / v.norm())
            assert rel < 4 * torch.finfo(g.dtype).eps, f"{name}: {rel:.3e}"


def step(dtype, case, seed, scale=None, mode=None, do_scale=1.0, **kw):
    n1, n2, d, dr, tokens, kv, m, packed, behind = CASES[case]
    mode = m if mode is None else mode
    scale = 1 / math.sqrt(d + dr) if scale is None else scale
    t = make(dtype, n1, n2, d, dr, tokens, kv, packed, seed, behind)
    do = make(dtype, n1, n1, d, 0, tokens, tokens, packed, seed + 1, behind)["query"] * do_scale
    fwd = call(t, tokens, kv, packed, scale, mode)
    return t, do, fwd, tokens, kv, packed, scale, mode


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_formula(dtype, case):
    t, do, fwd, tokens, kv, packed, scale, mode = step(dtype, case, 300 + case)
    got = gradients(t, do, fwd, tokens, kv, packed, scale, mode)
    check(got, exact_grads(t, do, tokens, kv, packed, scale, mode))
    again = gradients(t, do, fwd, tokens, kv, packed, scale, mode)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("splits", [1, 2, 5, 64])
@pytest.mark.parametrize("case", [4, 6, 7, 9, 10, 14])
def test_ranges(case, splits):
    t, do, fwd, tokens, kv, packed, scale, mode = step(BF, case, 400 + case)
    check(gradients(t, do, fwd, tokens, kv, packed, scale, mode, splits=splits),
          exact_grads(t, do, tokens, kv, packed, scale, mode))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.7])
def test_scales(dtype, scale):
    t, do, fwd, tokens, kv, packed, scale, mode = step(dtype, 6, 500, scale)
    check(gradients(t, do, fwd, tokens, kv, packed, scale, mode), exact_grads(t, do, tokens, kv, packed, scale, mode))


@pytest.mark.parametrize("do_scale", [2.0 ** -12, 2.0 ** 9])
def test_small_and_large_gradients_fp16(do_scale):
    """dS from 2^-26 on (which fp16 by itself would round to one or two bits), and past 65504."""
    t, do, fwd, tokens, kv, packed, scale, mode = step(HF, 12, 600, do_scale=do_scale)
    got = gradients(t, do, fwd, tokens, kv, packed, scale, mode)
    want = exact_grads(t, do, tokens, kv, packed, scale, mode)
    for name, g in zip(NAMES, got):
        if g is not None:
            v, tol = want[name]
            ok = v.abs() < 60000   # (what the output type holds)
            assert (((g.double() - v).abs() - tol)[ok] <= 0).all(), name


@pytest.mark.parametrize("how", ["fused", "odd", "heads first", "last"])
@pytest.mark.parametrize("packed", [True, False])
def test_strides(how, packed):
    tokens, kv = [80, 41], [95, 60]
    t = make(BF, 4, 2, 128, 64, tokens, kv, packed, 31)
    do = make(BF, 4, 4, 128, 0, tokens, tokens, packed, 32)["query"]
    fwd = call(t, tokens, kv, packed, 0.1)
    want = gradients(t, do, fwd, tokens, kv, packed, 0.1)
    got = gradients({k: strided(v, how) for k, v in t.items()}, strided(do, how), (strided(fwd[0], how),) + tuple(fwd[1:]), tokens,
                    kv, packed, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_shared_rotary_key_and_broadcast_gradient():
    t = make(BF, 6, 3, 128, 64, [70], [70], True, 33)
    t["key_rope"] = t["key_rope"][:, :1].expand(70, 3, 64)
    do = torch.ones(6, 128, dtype=BF, device="cuda").expand(70, 6, 128)   # of a sum over the rows
    fwd = call(t, [70], [70], True, 0.1)
    check(gradients(t, do, fwd, [70], [70], True, 0.1), exact_grads(t, do, [70], [70], True, 0.1))


def test_differences():
    """The directional derivative of sum(out d) along u, by differences of the formula in 64 bits at a step of 2^-10 (its
    error, some step^2, is below 1e-4 of the gradient's norm); the operator's gradient is off by its rounding, 4 eps."""
    t, do, fwd, tokens, kv, packed, scale, mode = step(BF, 8, 700)
    got = dict(zip(NAMES, gradients(t, do, fwd, tokens, kv, packed, scale, mode)))
    g, h = torch.Generator().manual_seed(5), 2.0 ** -10
    for what in ("query", "key", "value"):
        u = torch.randn(t[what].shape, generator=g).double().cuda()
        u = u / u.norm()
        f = lambda s: float((exact({**t, what: t[what].double() + s * u}, tokens, kv, packed, scale, mode)[0].reshape(do.shape) * do.double()).sum())
        d = got["d_" + what].double()
        assert abs((f(h) - f(-h)) / (2 * h) - float((d * u).sum())) < (1e-3 + 4 * torch.finfo(BF).eps) * float(d.norm())


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("what", ["query", "key", "value", "d_out"])
def test_values_that_are_not_finite(what, value):
    """They reach the gradients of what sees them, or is seen, and nothing else."""
    tokens, kv = [50, 200], [70, 200]
    t = make(BF, 4, 2, 128, 64, tokens, kv, False, 40, behind=3)
    t = {k: v.clone() for k, v in t.items()}
    do = make(BF, 4, 4, 128, 0, tokens, tokens, False, 41, behind=3)["query"].clone()
    clean = gradients(t, do, call(t, tokens, kv, False, 0.1), tokens, kv, False, 0.1)
    x = do if what == "d_out" else t[what]
    x[0, 70 if what in ("key", "value") else 50:] = value     # padding
    x[1, 150, 1] = value                     # query 150 of heads 1 and (keys) token 150 of the heads 2, 3
    got = gradients(t, do, call(t, tokens, kv, False, 0.1), tokens, kv, False, 0.1)
    queries = what in ("query", "d_out")
    for name, a, b in zip(NAMES, got, clean):
        assert torch.equal(a[0], b[0]), name
        assert not a[0, 50 if "query" in name else 70:].any() and not a[1, 200:].any(), name
        heads_q = [1] if queries else [2, 3]
        head_k = 0 if queries else 1
        if "query" in name:
            other = [h for h in range(4) if h not in heads_q]
            assert torch.equal(a[1][:, other], b[1][:, other]), name
            rows = [r for r in range(203) if r != 150] if queries else list(range(150)) + [200, 201, 202]
            assert torch.equal(a[1][rows], b[1][rows]), name
            assert not torch.isfinite(a[1, 150, heads_q]).all(), name
        else:
            assert torch.equal(a[1][:, 1 - head_k], b[1][:, 1 - head_k]), name
            if queries:   # what query 150 does not see
                assert torch.equal(a[1, 151:], b[1, 151:]), name
            assert not torch.isfinite(a[1, 150, head_k]).all() or what in ("key", "value"), name


def test_no_rows_no_keys():
    e = lambda *s: torch.ones(*s, dtype=BF, device="cuda")
    f = lambda *s: torch.zeros(*s, device="cuda")
    for q, k in ((e(0, 4, 64), e(7, 2, 64)), (e(5, 4, 64), e(0, 2, 64))):
        got = dsa.dense_attention_grad(q, k, k, q, q, f(2, q.shape[0], 2), f(2, q.shape[0], 2), layout="TND")
        assert got[0].shape == q.shape and got[1].shape == k.shape and not got[0].any() and not got[1].any() and not got[2].any()


def test_plan_on_another_stream_and_in_a_graph():
    tokens, kv = [100, 31, 257], [100, 60, 257]
    t = make(HF, 8, 2, 64, 0, tokens, kv, True, 50)
    do = make(HF, 8, 8, 64, 0, tokens, tokens, True, 51)["query"]
    fwd = dsa.DenseAttentionPlan(t["query"], t["key"], t["value"], 0.1, [100, 131, 388], [100, 160, 417], layout="TND",
                                 return_softmax_lse=True)
    out, mx, sm = fwd.run()
    bwd = dsa.DenseAttentionGradPlan(t["query"], t["key"], t["value"], do, out, mx, sm, 0.1, actual_seq_lengths_query=[100, 131, 388],
                                     actual_seq_lengths_kv=[100, 160, 417], layout="TND")
    want = gradients(t, do, (out, mx, sm), tokens, kv, True, 0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = bwd.run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fwd.run()
        got = bwd.run()
    for seed in (52, 53, 54):
        t2 = make(HF, 8, 2, 64, 0, tokens, kv, True, seed)
        do2 = make(HF, 8, 8, 64, 0, tokens, tokens, True, seed + 100)["query"]
        for k in ("query", "key", "value"):
            t[k].copy_(t2[k])
        do.copy_(do2)
        graph.replay()
        torch.cuda.synchronize()
        want = gradients(t2, do2, call(t2, tokens, kv, True, 0.1), tokens, kv, True, 0.1)
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, want))
