"""shared_prefix_attention against the formula in 64 bits.

Tolerances, per element, from w = the exact softmax weights and A = sum_t w_t |v_t|:
  * the output's rounding: half a step, eps / 2 of the value;
  * P is rounded to the io type before the product: eps / 2 of each term, eps / 2 * A in all;
  * scores are 32-bit sums of D + 64 products, off by at most ds = (D + 64) 2^-24 max_t sum_i |q_i k_i| scale:
    weights move by 2 ds relative, the output by 2 ds A; the exponential and the 32-bit sums of P and P v
    add 2^-20 A.
softmax_max is within ds, softmax_sum within ds + 2^-20 relative (twice ds: its max moves too)."""
import math

import pytest
import torch

import dsa_triton_ascend_amd as dsa

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def make(dtype, n1, d, tokens, kv, prefix, page, packed, seed, tail=0, extra_cols=0, spare=3):
    """Inputs on the GPU; every table row has its own pages, also for the prefix (only row 0's count)."""
    g = torch.Generator().manual_seed(seed)
    cols = max(1, -(-max(kv + [prefix]) // page)) + extra_cols
    blocks = len(kv) * cols + spare
    table = torch.randperm(blocks, generator=g)[:len(kv) * cols].int().view(len(kv), cols)
    lead = (sum(tokens) + tail,) if packed else (len(tokens), max(tokens))
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    return dict(q=r(*lead, n1, d), qr=r(*lead, n1, 64), k=r(blocks, page, 1, d), kr=r(blocks, page, 1, 64), table=table.cuda())


def exact(t, tokens, kv, prefix, scale, mode, packed):
    """(out, max, sum, tolerance of out, ds) in 64 bits; rows in packed order."""
    q, qr, table = t["q"], t["qr"], t["table"]
    n1, d = q.shape[-2:]
    blocks, page = t["k"].shape[:2]
    kc, krc = t["k"].double().view(-1, d), t["kr"].double().view(-1, 64)
    Q, R = q.double().reshape(-1, n1, d), qr.double().reshape(-1, n1, 64)
    out = torch.zeros(Q.shape, dtype=torch.float64, device="cuda")
    top, tot, ds = (torch.zeros(Q.shape[:2], dtype=torch.float64, device="cuda") for _ in range(3))
    A = torch.zeros_like(out)
    S = q.shape[0] if packed else q.shape[1]
    at = 0
    for b, (nq, nk) in enumerate(zip(tokens, kv)):
        r0 = at if packed else b * S
        at += nq
        pos = torch.arange(nk, device="cuda")
        row = torch.where(pos < prefix, 0, b)
        blk = table.long()[row, pos // page] if nk else pos
        ok = (blk >= 0) & (blk < blocks)
        phys = torch.where(ok, blk * page + pos % page, 0)
        K, KR = kc[phys] * ok[:, None], krc[phys] * ok[:, None]
        K, KR = torch.where(ok[:, None], K, 0.0), torch.where(ok[:, None], KR, 0.0)
        for s in range(nq):
            n = nk if mode == 0 else max(0, min(nk, nk - nq + s + 1))
            if n == 0:
                continue
            a, c = Q[r0 + s], R[r0 + s]
            sc = (a @ K[:n].t() + c @ KR[:n].t()) * scale
            m = sc.max(-1).values
            e = torch.exp(sc - m[:, None])
            out[r0 + s], top[r0 + s], tot[r0 + s] = (e @ K[:n]) / e.sum(-1, keepdim=True), m, e.sum(-1)
            A[r0 + s] = (e @ K[:n].abs()) / e.sum(-1, keepdim=True)
            ds[r0 + s] = (a.abs() @ K[:n].abs().t() + c.abs() @ KR[:n].abs().t()).max(-1).values * abs(scale) * (d + 64) * 2.0 ** -24
    eps = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * eps
    tol = eps * out.abs() + (eps + 2 * ds[..., None] + 2.0 ** -20) * A + tiny
    return out, top, tot, tol, ds


def check(got, want, stats=True, rows=None):
    out, top, tot, tol, ds = want
    sel = slice(None) if rows is None else rows
    o = got[0].double().reshape(out.shape)[sel]
    assert torch.isfinite(o).all()
    over = ((o - out[sel]).abs() - tol[sel]).max() if o.numel() else 0.0
    assert over <= 0, f"out over its bound by {float(over):.3e}"
    if stats:
        m, l = (x.double().reshape(top.shape)[sel] for x in got[1:])
        assert ((m - top[sel]).abs() <= ds[sel] + 1e-30).all()
        assert ((l - tot[sel]).abs() <= (2 * ds[sel] + 2.0 ** -20) * tot[sel]).all()


def call(t, tokens, kv, prefix, scale, mode, packed, **kw):
    cu = torch.tensor(tokens).cumsum(0).tolist() if packed else tokens
    return dsa.shared_prefix_attention(t["q"], t["k"], t["k"], t["table"], prefix, scale, cu, kv, t["qr"], t["kr"],
                                       layout_query="TND" if packed else "BSND", sparse_mode=mode,
                                       return_softmax_lse=True, **kw)


CASES = [  # n1, d, tokens, kv, prefix, page, mode, packed
    (1, 512, [1], [1], 0, 16, 3, False),
    (1, 128, [1], [1], 1, 1, 3, False),
    (16, 512, [1, 1, 1, 1], [305, 311, 340, 327], 304, 16, 3, False),
    (16, 512, [1] * 9, [700, 650, 901, 644, 700, 701, 702, 1200, 643], 643, 64, 3, False),
    (128, 512, [1, 1, 1], [513, 530, 777], 500, 128, 3, False),
    (32, 256, [2, 2, 2], [200, 260, 203], 199, 7, 3, False),
    (64, 512, [3, 1, 2], [163, 161, 290], 160, 48, 3, False),          # fewer queries than S
    (8, 128, [4, 4, 4, 4, 4], [40, 33, 97, 36, 64], 32, 32, 0, False),
    (64, 512, [40, 7, 90], [300, 263, 400], 256, 64, 3, True),           # prompts behind a document
    (128, 256, [33, 64], [33, 64], 0, 64, 3, True),                      # no prefix: causal prompts
    (4, 512, [5, 0, 17], [20, 30, 17], 9, 16, 3, True),                  # a sequence without queries
    (16, 512, [1, 1, 1, 1], [90, 0, 17, 300], 128, 16, 3, False),        # lengths inside the prefix, and none
    (32, 512, [6, 6], [4, 70], 2, 16, 3, False),                         # more queries than tokens: empty rows
    (2, 512, [130], [131], 64, 33, 3, True),
    (128, 512, [2, 2], [2500, 1300], 1027, 64, 0, False),
    (16, 128, [1] * 40, list(range(2100, 2140)), 2048, 128, 3, False),
    (16, 128, [900] + [1, 0, 2] * 20, [1100] + [205, 201, 260] * 20, 200, 64, 3, True),   # one long prompt, many short
    (128, 256, [0, 3, 150, 0, 0, 1, 0], [40, 50, 170, 33, 0, 41, 60], 33, 16, 3, True),  # rows packed between empty sequences
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_formula(dtype, case):
    n1, d, tokens, kv, prefix, page, mode, packed = CASES[case]
    t = make(dtype, n1, d, tokens, kv, prefix, page, packed, 100 + case, tail=3 if packed else 0)
    scale = 1 / math.sqrt(d + 64)
    want = exact(t, tokens, kv, prefix, scale, mode, packed)
    check(call(t, tokens, kv, prefix, scale, mode, packed), want)


@pytest.mark.parametrize("tokens,tail", [([1200, 3, 5], 700), ([3, 5, 1200], 700), ([900], 1), ([0, 0, 40], 300), ([2, 0], 90)])
def test_rows_behind_the_last_sequence_are_zeros(tokens, tail):
    """Many rows behind the last sequence, of one range (no join): evenly split and numbered-through items."""
    kv = [max(t, 1) for t in tokens]
    t = make(BF, 64, 128, tokens, kv, 0, 16, True, 300, tail=tail)
    for splits in (1, 3):
        with torch.no_grad():
            junk = torch.full((sum(tokens) + tail + 8, 64, 128), float("nan"), dtype=BF, device="cuda")   # what the output's memory held
        del junk
        check(call(t, tokens, kv, 0, 0.07, 3, True, kv_splits=splits), exact(t, tokens, kv, 0, 0.07, 3, True))


@pytest.mark.parametrize("splits", [1, 2, 5, 64])
@pytest.mark.parametrize("case", [3, 6, 8, 9, 11, 14])
def test_forced_splits(splits, case):
    n1, d, tokens, kv, prefix, page, mode, packed = CASES[case]
    t = make(BF, n1, d, tokens, kv, prefix, page, packed, 200 + case, tail=3 if packed else 0)
    want = exact(t, tokens, kv, prefix, 0.05, mode, packed)
    check(call(t, tokens, kv, prefix, 0.05, mode, packed, kv_splits=splits), want)


@pytest.mark.parametrize("splits", [3, 5, 7, 11])
def test_prefix_items_over_the_xcds(splits):
    """Numbers of prefix items that eight does not divide, the last tile with rows of one wave only (816 head rows)."""
    kv = [701 + b % 60 for b in range(51)]
    t = make(BF, 16, 128, [1] * 51, kv, 700, 64, False, 400)
    check(call(t, [1] * 51, kv, 700, 0.05, 3, False, kv_splits=splits), exact(t, [1] * 51, kv, 700, 0.05, 3, False))


@pytest.mark.parametrize("n1", [1, 2, 4, 8, 16, 32, 64, 128])
@pytest.mark.parametrize("d", [128, 256, 512])
def test_head_counts(n1, d):
    tokens, kv = [2, 2, 2], [100, 117, 150]
    t = make(HF, n1, d, tokens, kv, 96, 32, False, 7)
    check(call(t, tokens, kv, 96, 0.04, 3, False), exact(t, tokens, kv, 96, 0.04, 3, False))


@pytest.mark.parametrize("prefix", [0, 300])
def test_missing_blocks_read_zero_rows(prefix):
    tokens, kv = [2, 1, 2], [400, 333, 390]
    t = make(BF, 16, 512, tokens, kv, prefix, 16, False, 8)
    t["table"][0, 3], t["table"][1, 20], t["table"][2, 21] = -1, t["k"].shape[0], 2 ** 31 - 1
    check(call(t, tokens, kv, prefix, 0.04, 3, False), exact(t, tokens, kv, prefix, 0.04, 3, False))


@pytest.mark.parametrize("scale", [-0.04, 0.0, 0.4, -1.5])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_scales(scale, dtype):
    """Negative and zero scales, and scores of up to +-100: the reference maximum moves, rows are rescaled."""
    tokens, kv = [3, 3], [500, 640]
    for n1 in (8, 128):
        t = make(dtype, n1, 512, tokens, kv, 480, 32, False, 9)
        check(call(t, tokens, kv, 480, scale, 3, False), exact(t, tokens, kv, 480, scale, 3, False))


def test_rising_scores():
    """Each tile's maximum exceeds the last one's by more than the lazy threshold: rescales in every tile."""
    tokens, kv = [1, 1], [330, 400]
    for dtype in (BF, HF):
        t = make(dtype, 64, 512, tokens, kv, 300, 50, False, 10)
        order = torch.cat([t["table"][0].long(), t["table"][1].long()])
        k = t["k"].view(t["k"].shape[0], 50, 512)
        k[order, :, 0] = torch.linspace(-20, 60, order.numel() * 50).view(-1, 50).to(dtype).cuda()
        t["q"][..., 0] = 4.0
        check(call(t, tokens, kv, 300, 0.9, 3, False), exact(t, tokens, kv, 300, 0.9, 3, False))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n1", [8, 64, 128])
def test_values_that_no_row_sees(value, n1):
    """Cache slots behind the lengths, tokens of the prefix behind a short sequence's end, later tokens of
    a causal step, queries behind a sequence's count: what is not finite there reaches no other row."""
    tokens, kv, prefix, page = [5, 2, 5], [230, 100, 219], 170, 32
    t = make(BF, n1, 512, tokens, kv, prefix, page, False, 11)
    want = exact(t, tokens, kv, prefix, 0.04, 3, False)
    t["q"][1, 2:] = value
    t["qr"][1, 2:] = value
    k, kr, tab = t["k"], t["kr"], t["table"].long()
    for b in range(3):                        # behind each sequence
        for p in range(kv[b], tab.shape[1] * page):
            k[tab[b, p // page], p % page] = value
            kr[tab[b, p // page], p % page] = value
    check(call(t, tokens, kv, prefix, 0.04, 3, False), want)
    # the last two tokens of sequence 0, that its first rows do not see; a prefix token behind sequence 1's end
    for b, p in ((0, 229), (0, 228), (0, 150)):
        k[tab[b, p // page], p % page, 0, 7] = value
        kr[tab[b, p // page], p % page, 0, 3] = value
    got = call(t, tokens, kv, prefix, 0.04, 3, False)
    check(got, want, rows=slice(5, 7))       # sequence 1: 100 tokens, none of them touched
    # token 150 is everyone else's: the formula gives NaN where its value is not finite (0 x inf where the
    # score is -inf), and in the whole row where the score is NaN or +inf
    assert torch.isnan(got[0][2, ..., 7]).all() and torch.isnan(got[0][0, ..., 7]).all()
    if math.isnan(value):
        assert torch.isnan(got[0][2]).all() and torch.isnan(got[0][0]).all()
    k[tab[0, 150 // page], 150 % page, 0, 7] = 0
    kr[tab[0, 150 // page], 150 % page, 0, 3] = 0
    want = exact({**t, "k": torch.nan_to_num(k, 0, 0, 0), "kr": torch.nan_to_num(kr, 0, 0, 0)}, tokens, kv, prefix, 0.04, 3, False)
    got = call(t, tokens, kv, prefix, 0.04, 3, False)
    check(got, want, rows=slice(0, 3))       # rows 0 to 2 of sequence 0 see neither 228 nor 229
    assert torch.isnan(got[0][0, 3:, :, 7]).all()
    check(got, want, rows=slice(10, 15))


def test_equals_sparse_attention_over_all_tokens():
    """The same rows through sparse_flash_attention with every visible token selected: two kernels of the
    package agree within both their roundings."""
    tokens, kv, prefix, page, n1 = [4, 4], [120, 90], 80, 16, 32
    t = make(BF, n1, 512, tokens, kv, prefix, page, False, 12)
    t["table"][1, :prefix // page] = t["table"][0, :prefix // page]
    si = torch.full((2, 4, 1, 128), -1, dtype=torch.int32)
    for b in range(2):
        for s in range(4):
            n = kv[b] - 4 + s + 1
            si[b, s, 0, :n] = torch.arange(n)
    ref = dsa.sparse_flash_attention(t["q"], t["k"], t["k"], si.cuda(), 0.04, t["table"], None, kv, t["qr"], t["kr"],
                                     layout_kv="PA_BSND", sparse_mode=3, return_softmax_lse=True)
    got = call(t, tokens, kv, prefix, 0.04, 3, False)
    out, _, _, tol, ds = exact(t, tokens, kv, prefix, 0.04, 3, False)
    assert ((got[0].double() - ref[0].double()).reshape(out.shape).abs() <= 2 * tol).all()
    assert torch.allclose(got[1], ref[1], atol=2e-5) and torch.allclose(got[2], ref[2], rtol=2e-4)


def test_far_blocks():
    """Blocks past 2^32 bytes of the cache."""
    t = make(BF, 16, 512, [1], [100], 64, 64, False, 13)
    k = torch.zeros(70000, 64, 1, 512, dtype=BF, device="cuda")
    kr = torch.zeros(70000, 64, 1, 64, dtype=BF, device="cuda")
    want = exact(t, [1], [100], 64, 0.04, 3, False)
    far = torch.tensor([[69999, 66001]], dtype=torch.int32, device="cuda")
    k[far[0].long()], kr[far[0].long()] = t["k"][t["table"][0].long()], t["kr"][t["table"][0].long()]
    check(call({**t, "k": k, "kr": kr, "table": far}, [1], [100], 64, 0.04, 3, False), want)


@pytest.mark.parametrize("n1", [16, 128])
def test_plan_streams_and_graphs(n1):
    """A plan built on one stream runs on another; a captured run() reads act_k and the table on the
    device: lengths that grow past the plan's own, two graphs of two plans, each replayed."""
    tokens, kv, prefix = [1] * 6, [210, 230, 0, 201, 250, 300], 200
    t = make(BF, n1, 512, tokens, kv, prefix, 16, False, 14, extra_cols=8)
    args = (t["q"], t["k"], t["k"], t["table"], prefix, 0.04, None)
    kw = dict(query_rope=t["qr"], key_rope=t["kr"], return_softmax_lse=True)
    build, use = torch.cuda.Stream(), torch.cuda.Stream()
    build.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(build):
        plan = dsa.SharedPrefixPlan(*args, kv, **kw)
        other = dsa.SharedPrefixPlan(*args, [v + 5 for v in kv], **kw)
    use.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(use):
        got = plan.run()
    use.synchronize()
    check(got, exact(t, tokens, kv, prefix, 0.04, 3, False))
    graphs = []
    for p in (plan, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p.run()
        graphs.append(graph)
    for step in (1, 2, 90):
        lens = [v + step for v in kv]
        plan.act_k[:6].copy_(torch.tensor(lens, dtype=torch.int32))
        t["q"].copy_(torch.randn_like(t["q"].float()).to(BF))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        check((plan.out, plan.sm[0], plan.sm[1]), exact(t, tokens, lens, prefix, 0.04, 3, False))
        check((other.out, other.sm[0], other.sm[1]), exact(t, tokens, [v + 5 for v in kv], prefix, 0.04, 3, False))
        eager = dsa.SharedPrefixPlan(*args, [v + 5 for v in kv], **kw).run()
        assert torch.equal(eager[0], other.out)          # the same bits in every run


def test_strided_inputs_and_defaults():
    t = make(BF, 16, 512, [2, 2], [96, 96], 48, 48, False, 15)
    buf = torch.zeros(2, 2, 16, 577, dtype=BF, device="cuda")
    buf[..., 1:513], buf[..., 513:] = t["q"], t["qr"]
    want = exact(t, [2, 2], [96, 96], 48, 0.04, 3, False)
    m = dsa.SharedPrefixAttention(0.04, return_softmax_lse=True)
    got = m(buf[..., 1:513], t["k"], t["k"], t["table"].long(), 48, buf[..., 513:], t["kr"])
    check(got, want)
    out, mx, sm = dsa.shared_prefix_attention(t["q"], t["k"], t["k"], t["table"], 48, 0.04, query_rope=t["qr"], key_rope=t["kr"])
    assert torch.equal(out, got[0]) and not mx.any() and not sm.any() and mx.shape == (2, 1, 2, 16)
    empty = dsa.shared_prefix_attention(t["q"][:0], t["k"], t["k"], t["table"][:0], 48, 0.04, query_rope=t["qr"][:0], key_rope=t["kr"])
    assert empty[0].shape == (0, 2, 16, 512)
    none = dsa.shared_prefix_attention(t["q"], t["k"][:0], t["k"][:0], t["table"], 0, 0.04, None, [0, 0], t["qr"], t["kr"][:0])
    assert not none[0].any()


def test_append_then_attend():
    """As a serving loop uses them: a document appended once, its blocks shared by the table's rows, then
    steps of appended tokens with rotated queries, against dense attention over everything in 64 bits."""
    g = torch.Generator().manual_seed(16)
    B, N, page, P = 3, 16, 16, 70
    dev, f = "cuda", (1.0 / 10000 ** (torch.arange(32) / 32)).cuda()
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF).to(dev)
    blocks = 24
    k, kr = torch.zeros(blocks, page, 1, 512, dtype=BF, device=dev), torch.zeros(blocks, page, 1, 64, dtype=BF, device=dev)
    order = torch.randperm(blocks, generator=g).int()
    shared = order[:5]                                    # 70 tokens: the fifth block is part full
    table = torch.cat([shared[:4].expand(B, 4), order[5:5 + 4 * B].view(B, 4)], 1).contiguous()
    table[0, 4] = shared[4]
    table = table.to(dev)
    w = torch.ones(512, device=dev)
    doc = (rnd(1, P, 1, 512), rnd(1, P, 1, 64))
    dsa.latent_cache_append(*doc, k, kr, table[:1], f, [P], norm_weight=w)
    part = P % page
    for b in (1, 2):                                      # each sequence continues in its own copy of that block
        k[table[b, 4].long(), :part], kr[table[b, 4].long(), :part] = k[shared[4].long(), :part], kr[shared[4].long(), :part]
    lens = [P, P, P]
    for step, nq in enumerate(([3, 1, 2], [1, 1, 1], [2, 0, 3])):
        lens = [a + n for a, n in zip(lens, nq)]
        cu = torch.tensor(nq).cumsum(0).tolist()
        T = sum(nq)
        dsa.latent_cache_append(rnd(T, 1, 512), rnd(T, 1, 64), k, kr, table, f, lens, cu, norm_weight=w, layout="TND")
        pos = torch.cat([torch.arange(a - n, a) for a, n in zip(lens, nq)]).to(dev)
        q, qr = rnd(T, N, 512), dsa.rotary_embedding(rnd(T, N, 64), pos, f, layout="TND")
        t = dict(q=q, qr=qr, k=k, kr=kr, table=table)
        check(call(t, nq, lens, P, 0.04, 3, True), exact(t, nq, lens, P, 0.04, 3, True))
        check(call(t, nq, lens, 0, 0.04, 3, True), exact(t, nq, lens, 0, 0.04, 3, True))   # the rows' own tables agree
        a, b_ = (call(t, nq, lens, p, 0.04, 3, True)[0].double() for p in (P, 0))
        assert float((a - b_).abs().max()) < 2 ** -6 * float(a.abs().max())


@pytest.mark.parametrize("n1", [8, 32, 128])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_scales_that_are_not_finite(scale, n1):
    """The formula's scores are NaN or of infinite size then, and so no row that sees a token has a finite value; rows
    that see none stay zeros."""
    tokens, kv = [2, 2], [300, 1]
    t = make(BF, n1, 128, tokens, kv, 200, 32, False, 17)
    for splits in (1, 3):
        out, _, total = call(t, tokens, kv, 200, scale, 3, False, kv_splits=splits)
        seen = torch.tensor([[True, True], [False, True]])
        assert torch.isnan(out[seen.cuda()]).all() and not out[1, 0].any()
        assert not torch.isfinite(total.reshape(2, 2, n1)[0]).any() and not total.reshape(2, 2, n1)[1, 0].any()


def test_packed_without_lengths_is_one_sequence():
    t = make(BF, 16, 128, [37], [300], 0, 32, True, 18)
    kw = dict(actual_seq_lengths_kv=[300], query_rope=t["qr"], key_rope=t["kr"], layout_query="TND", return_softmax_lse=True)
    got = dsa.shared_prefix_attention(t["q"], t["k"], t["k"], t["table"], 0, 0.05, **kw)
    check(got, exact(t, [37], [300], 0, 0.05, 3, True))


@pytest.mark.parametrize("gap", [10.0, 15.0, 17.5, 20.0])
@pytest.mark.parametrize("n1", [16, 64, 128])
def test_small_weights_of_many_tokens(n1, gap):
    """One token whose score is `gap` above those of 60,000 others: together their weights (4.5e-5 to 2.1e-9 each) are
    seen in the columns where the one is zero. A weight below fp16's normal numbers is off by half of its smallest
    step, 2^-25, where the row's largest is e^6 or more: 60,001 of them by 4.4e-6 at most, beside the usual bound."""
    kv, page = 60001, 512
    t = make(HF, n1, 128, [1], [kv], 0, page, False, 19)
    k = t["k"]
    k.zero_()
    t["kr"].zero_()
    t["q"].zero_()
    t["q"][..., 0] = 1.0
    k[..., 1:] = 1.0
    at = 777
    k[t["table"][0, at // page].long(), at % page, 0, 0] = gap
    k[t["table"][0, at // page].long(), at % page, 0, 1:] = 0.0
    for splits in (1, 0):
        want = list(exact(t, [1], [kv], 0, 1.0, 3, False))
        want[3] = want[3] + kv * 2.0 ** -25 * math.exp(-6)
        check(call(t, [1], [kv], 0, 1.0, 3, False, kv_splits=splits), want)
