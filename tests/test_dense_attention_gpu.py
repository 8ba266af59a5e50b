"""dense_attention against the formula in 64 bits.

Tolerances, per element, from w = the exact softmax weights and A = sum_t w_t |v_t|:
  * the output's rounding: half a step, eps / 2 of the value;
  * P is rounded to the io type before the product: eps / 2 of each term, eps / 2 * A in all; fp16 rounds small ones to
    steps of 2^-24 where the row's largest is at least e^(6 - 10.5): half a step, 2^-25 e^4.5 / sum of each term;
  * scores are 32-bit sums of D + 64 products, off by at most ds = (D + 64) 2^-24 max_t sum_i |q_i k_i| scale: weights
    move by 2 ds relative, the output by 2 ds A; the exponential and the 32-bit sums of P and P v add 2^-20 A.
softmax_max is within ds, softmax_sum within 2 ds + 2^-20 relative (its max moves too)."""
import math

import pytest
import torch

import dsa_triton_ascend_amd as dsa

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def make(dtype, n1, n2, d, dr, tokens, kv, packed, seed, behind=0, q_scale=1.0):
    """Inputs on the GPU; padded and trailing rows hold values as well."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    lead = lambda n: (sum(n) + behind,) if packed else (len(n), max(n) + behind)
    ql, kl = lead(tokens), lead(kv)
    t = dict(query=r(*ql, n1, d) * q_scale, key=r(*kl, n2, d), value=r(*kl, n2, d), query_rope=None, key_rope=None)
    if dr:
        t.update(query_rope=r(*ql, n1, dr), key_rope=r(*kl, n2, dr))
    return t


def call(t, tokens, kv, packed, scale, mode=3, lse=True, **kw):
    cu = (lambda n: torch.tensor(n).cumsum(0).tolist()) if packed else (lambda n: n)
    return dsa.dense_attention(t["query"], t["key"], t["value"], scale, cu(tokens), cu(kv), t["query_rope"], t["key_rope"],
                               "TND" if packed else "BSND", mode, lse, **kw)


def exact(t, tokens, kv, packed, scale, mode=3):
    """(out, max, sum, tolerance of out, ds) in 64 bits, rows in packed order; statistics [rows, N1]."""
    cat = lambda a, b: a if b is None else torch.cat([a, b], -1)
    q, k, v = cat(t["query"], t["query_rope"]).double(), cat(t["key"], t["key_rope"]).double(), t["value"].double()
    S1, S2 = (0, 0) if packed else (q.shape[1], k.shape[1])
    q, k, v = (x if packed else x.flatten(0, 1) for x in (q, k, v))
    n1, n2, d = q.shape[1], k.shape[1], v.shape[-1]
    out = torch.zeros(q.shape[0], n1, d, dtype=torch.float64, device="cuda")
    A, (top, tot, ds) = torch.zeros_like(out), torch.zeros(3, q.shape[0], n1, dtype=torch.float64, device="cuda").unbind(0)
    fine = torch.zeros_like(top)
    aq, ak = 0, 0
    for b, (nq, nk) in enumerate(zip(tokens, kv)):
        r0, k0 = (aq, ak) if packed else (b * S1, b * S2)
        aq, ak = aq + nq, ak + nk
        if not nq or not nk:
            continue
        rows = slice(r0, r0 + nq)
        kk, vv = (x[k0:k0 + nk].repeat_interleave(n1 // n2, 1).transpose(0, 1) for x in (k, v))   # [N1, nk, .]
        qq = q[rows].transpose(0, 1)
        s = qq @ kk.transpose(1, 2) * scale
        seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda") if mode == 0 else \
            torch.ones(nq, nk, dtype=torch.bool, device="cuda").tril(nk - nq)
        s = s.masked_fill(~seen, -math.inf)
        live = seen.any(-1)
        m = s.amax(-1).masked_fill(~live, 0.0)
        e = torch.exp(s - m[..., None])
        l = e.sum(-1)
        w = e / l.masked_fill(~live, 1.0)[..., None]
        out[rows], A[rows] = (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1)
        top[rows], tot[rows] = m.transpose(0, 1), l.transpose(0, 1)
        mag = (qq.abs() @ kk.abs().transpose(1, 2)).masked_fill(~seen, 0.0).amax(-1)
        ds[rows] = mag.transpose(0, 1) * abs(scale) * q.shape[-1] * 2.0 ** -24
        fine[rows] = (2.0 ** -25 * math.exp(4.5) / l.masked_fill(~live, 1.0)).transpose(0, 1) * seen.sum(-1)[:, None]
    eps = torch.finfo(t["query"].dtype).eps / 2
    tiny = torch.finfo(t["query"].dtype).smallest_normal * eps
    small = fine[..., None] * v.abs().max() if t["query"].dtype == HF else 0.0
    return out, top, tot, eps * out.abs() + (eps + 2 * ds[..., None] + 2.0 ** -20) * A + small + tiny, ds


def rows_of(stat, packed):
    """[B,N2,S,G] or [N2,T,G] as [rows, N1]"""
    return stat.movedim(-3, -2).flatten(-2) if packed else stat.movedim(-3, -2).flatten(0, 1).flatten(-2)


def check(got, want, packed):
    out, top, tot, tol, ds = want
    o = got[0].double().reshape(out.shape)
    assert torch.isfinite(o).all()
    over = ((o - out).abs() - tol).max()
    assert over <= 0, f"out over its bound by {float(over):.3e}"
    m, l = (rows_of(x.double(), packed) for x in got[1:])
    assert ((m - top).abs() <= ds + 1e-30).all()
    assert ((l - tot).abs() <= (2 * ds + 2.0 ** -20) * tot).all()


CASES = [  # n1, n2, d, dr, tokens, kv, mode, packed, behind
    (1, 1, 64, 0, [1], [1], 3, True, 0),
    (8, 2, 64, 0, [60], [60], 3, True, 0),
    (6, 2, 128, 0, [33], [33], 3, True, 3),
    (4, 4, 128, 64, [129], [129], 3, True, 0),
    (5, 1, 128, 0, [70, 1, 64, 0, 200], [70, 1, 64, 9, 200], 3, True, 5),       # a group of five, a sequence without queries
    (3, 3, 64, 0, [100, 31, 65], [100, 31, 65], 0, False, 0),                    # padded, no causal mask
    (8, 4, 128, 64, [10, 64, 3], [50, 64, 300], 3, False, 2),                    # padded chunks after earlier keys
    (32, 4, 128, 0, [1, 1, 1], [500, 1, 1333], 3, False, 0),                     # single tokens
    (16, 1, 64, 0, [2, 2], [700, 333], 3, False, 0),
    (48, 2, 128, 64, [1], [4001], 3, True, 0),
    (2, 2, 128, 0, [70, 8], [30, 4], 3, True, 0),                                # more queries than keys: empty rows
    (2, 1, 64, 0, [5, 7], [0, 9], 3, True, 0),                                   # no keys
    (8, 8, 128, 0, [257, 511], [257, 511], 3, True, 1),
    (4, 2, 64, 0, [1025], [1025], 0, True, 0),
    (2, 2, 128, 64, [300], [1500], 3, True, 0),
    (4, 1, 128, 0, [1] * 30 + [900], [50] * 30 + [900], 3, True, 2),             # numbered through: one long, many short
    (128, 128, 64, 0, [140], [140], 3, True, 0),
    (128, 1, 128, 0, [9, 30], [40, 30], 3, True, 0),                             # 128 heads of one key head
    (16, 16, 128, 0, [2300, 2100], [2300, 2100], 3, True, 0),                    # 256 rows a work-group
    (16, 16, 64, 0, [2300, 2100], [2500, 2100], 3, False, 0),
    (16, 16, 128, 64, [4200], [4200], 3, True, 0),
    (12, 4, 128, 0, [3000], [3001], 0, True, 0),
    (16, 16, 64, 0, [2300, 2100], [4700, 2100], 3, False, 0),                    # the same after as many earlier tokens
    (32, 8, 64, 0, [1400], [1401], 0, True, 0),
    (32, 8, 128, 0, [1400], [2900], 3, True, 3),
    (12, 2, 128, 64, [2], [511], 3, True, 0),                                    # one range, then several
    (12, 2, 128, 64, [2], [512], 3, True, 0),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_formula(dtype, case):
    n1, n2, d, dr, tokens, kv, mode, packed, behind = CASES[case]
    t = make(dtype, n1, n2, d, dr, tokens, kv, packed, 100 + case, behind)
    scale = 1 / math.sqrt(d + dr)
    got = call(t, tokens, kv, packed, scale, mode)
    check(got, exact(t, tokens, kv, packed, scale, mode), packed)
    again = call(t, tokens, kv, packed, scale, mode, lse=False)
    assert torch.equal(again[0], got[0]) and not again[1].any() and not again[2].any()


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
@pytest.mark.parametrize("case", [4, 6, 7, 9, 10, 14])
def test_ranges_of_tokens(case, splits):
    n1, n2, d, dr, tokens, kv, mode, packed, behind = CASES[case]
    t = make(BF, n1, n2, d, dr, tokens, kv, packed, 200 + case, behind)
    check(call(t, tokens, kv, packed, 0.1, mode, kv_splits=splits), exact(t, tokens, kv, packed, 0.1, mode), packed)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 2.0])
def test_scales(scale):
    t = make(BF, 4, 2, 128, 64, [90, 33], [90, 70], True, 5)
    check(call(t, [90, 33], [90, 70], True, scale), exact(t, [90, 33], [90, 70], True, scale), True)
    bad = call(t, [90, 33], [90, 70], True, math.nan)
    assert bad[0].isnan().all() and bad[2].isnan().all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_growing_and_sharp_scores(dtype):
    """Maxima that move from tile to tile, and weights from 1 down to nothing."""
    t = make(dtype, 2, 1, 128, 0, [300], [300], True, 8, q_scale=4.0)
    t["key"] *= torch.linspace(0.2, 4.0, 300, device="cuda").to(dtype)[:, None, None]
    check(call(t, [300], [300], True, 0.3), exact(t, [300], [300], True, 0.3), True)
    t["key"] = t["key"].flip(0).contiguous()
    check(call(t, [300], [300], True, 0.3), exact(t, [300], [300], True, 0.3), True)


def test_many_small_weights_fp16():
    """One token 9 above 30,000 others that add up to more than it."""
    t = make(HF, 1, 1, 64, 0, [1], [30000], True, 3)
    t["query"][:], t["key"][:] = 0.0, 0.0
    t["query"][..., 0], t["key"][17, 0, 0] = 1.0, 9.0
    check(call(t, [1], [30000], True, 1.0), exact(t, [1], [30000], True, 1.0), True)
    check(call(t, [1], [30000], True, 1.0, kv_splits=1), exact(t, [1], [30000], True, 1.0), True)


def strided(x, how):
    if how == "fused":          # a slice of wider heads
        y = torch.zeros(*x.shape[:-1], x.shape[-1] + 72, dtype=x.dtype, device=x.device)[..., 8:8 + x.shape[-1]]
    elif how == "odd":          # heads off 16-byte borders: copied
        y = torch.zeros(*x.shape[:-1], x.shape[-1] + 3, dtype=x.dtype, device=x.device)[..., 1:1 + x.shape[-1]]
    elif how == "heads first":  # [heads, rows, width] underneath
        y = torch.zeros(x.shape[-2], *x.shape[:-2], x.shape[-1], dtype=x.dtype, device=x.device).movedim(0, -2)
    else:                       # last dimension strided: copied
        y = torch.zeros(*x.shape[:-1], x.shape[-1] * 2, dtype=x.dtype, device=x.device)[..., ::2]
    return y.copy_(x)


@pytest.mark.parametrize("how", ["fused", "odd", "heads first", "last"])
@pytest.mark.parametrize("packed", [True, False])
def test_strides(how, packed):
    tokens, kv = [80, 41], [95, 60]
    t = make(BF, 4, 2, 128, 64, tokens, kv, packed, 31)
    want = call(t, tokens, kv, packed, 0.1)
    got = call({k: strided(v, how) for k, v in t.items()}, tokens, kv, packed, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_one_rotary_key_for_all_heads():
    t = make(BF, 8, 8, 128, 64, [130], [130], True, 32)
    one = t["key_rope"][:, :1]
    t["key_rope"] = one.expand(130, 8, 64)
    got = call(t, [130], [130], True, 0.1)
    t["key_rope"] = one.repeat(1, 8, 1)
    assert all(torch.equal(a, b) for a, b in zip(got, call(t, [130], [130], True, 0.1)))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("mode", [0, 3])
def test_values_that_are_not_finite(what, value, mode):
    """Padding, rows behind, other sequences and later tokens: rows that do not see them are not affected."""
    tokens, kv = [50, 200], [70, 200]
    t = make(BF, 4, 2, 128, 0, tokens, kv, False, 40, behind=3)
    t["query"] = t["query"].clone()
    want = call(t, tokens, kv, False, 0.1, mode)
    t[what][0, 70:] = value                 # behind the first sequence's keys
    t["query"][0, 50:] = value
    t[what][1, 150, 1] = value              # a token that queries 150 .. 199 of the second see
    got = call(t, tokens, kv, False, 0.1, mode)
    first = 150 if mode == 3 else 0
    assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[0][1, :first], want[0][1, :first])
    assert torch.equal(got[0][1, :, :2], want[0][1, :, :2])       # the other key head's queries
    if value != value or what == "value":
        assert not torch.isfinite(got[0][1, first:200, 2:]).all(-1).any()
    assert not got[0][0, 50:].any() and not got[0][1, 200:].any()


@pytest.mark.parametrize("d,dr,mode", [(64, 0, 0), (128, 0, 0), (128, 0, 3), (128, 64, 0), (128, 64, 3)])
def test_values_that_are_not_finite_in_wide_work_groups(d, dr, mode):
    tokens = [1400, 900]
    t = make(BF, 32, 8, d, dr, tokens, tokens, False, 41)
    want = call(t, tokens, tokens, False, 0.1, mode)
    t["value"][1, 333, 1] = math.inf
    t["key"][1, 900:], t["value"][1, 900:], t["query"][1, 900:] = math.nan, math.nan, math.inf
    got = call(t, tokens, tokens, False, 0.1, mode)
    first = 333 if mode == 3 else 0
    assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[0][1, :first], want[0][1, :first])
    assert torch.equal(got[0][1, :, :4], want[0][1, :, :4]) and torch.equal(got[0][1, :, 8:], want[0][1, :, 8:])
    assert not torch.isfinite(got[0][1, first:900, 4:8]).all(-1).any() and not got[0][1, 900:].any()


def test_no_rows_no_keys():
    e = lambda *s: torch.empty(*s, dtype=BF, device="cuda")
    out, mx, sm = dsa.dense_attention(e(0, 4, 64), e(7, 2, 64), e(7, 2, 64), layout="TND", return_softmax_lse=True)
    assert out.shape == (0, 4, 64) and mx.shape == (2, 0, 2)
    for layout, q, k in (("TND", e(5, 4, 64), e(0, 2, 64)), ("BSND", e(2, 5, 4, 64), e(2, 0, 2, 64)), ("BSND", e(0, 5, 4, 64), e(0, 3, 2, 64))):
        out, mx, sm = dsa.dense_attention(q, k, k, layout=layout, return_softmax_lse=True)
        assert out.shape == q.shape and not out.any() and not mx.any() and not sm.any()


def test_plan_on_another_stream_and_in_a_graph():
    tokens, kv = [1, 1, 1], [900, 1400, 333]
    t = make(BF, 16, 2, 128, 0, tokens, kv, False, 50)
    plan = dsa.DenseAttentionPlan(t["query"], t["key"], t["value"], 0.1, tokens, kv, return_softmax_lse=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [x.clone() for x in plan.run()]
    torch.cuda.current_stream().wait_stream(s)
    want = call(t, tokens, kv, False, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = plan.run()
        once = dsa.dense_attention(t["query"], t["key"], t["value"], 0.1, tokens, kv)   # its lengths become part of the graph
    for seed in (51, 52, 53):
        t2 = make(BF, 16, 2, 128, 0, tokens, kv, False, seed)
        for k in ("query", "key", "value"):
            t[k].copy_(t2[k])
        graph.replay()
        torch.cuda.synchronize()
        want = call(t2, tokens, kv, False, 0.1)
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(once[0], want[0])


def test_rows_far_apart():
    """Key rows 2^23 elements from each other: byte offsets past 2^32."""
    n = 300
    wide = torch.empty(n, 1 << 23, dtype=BF, device="cuda")
    t = make(BF, 2, 1, 128, 0, [n], [n], True, 60)
    want = call(t, [n], [n], True, 0.1)
    for what, at in (("key", 0), ("value", 1024)):
        far = wide[:, at:at + 128].unsqueeze(1)
        far.copy_(t[what])
        t[what] = far
    got = call(t, [n], [n], True, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_module():
    t = make(BF, 4, 2, 64, 0, [20, 9], [20, 9], False, 70)
    m = dsa.DenseAttention(0.2, return_softmax_lse=True)
    got = m(t["query"], t["key"], t["value"], actual_seq_lengths_query=[20, 9], actual_seq_lengths_kv=[20, 9])
    assert all(torch.equal(a, b) for a, b in zip(got, call(t, [20, 9], [20, 9], False, 0.2)))
