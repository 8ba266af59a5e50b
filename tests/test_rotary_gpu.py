"""Rotary positions and the appends to the paged caches against 64-bit forms, at the sizes, strides
and lengths where they can go wrong, then the whole chain: append, indexer, sparse attention.

Tolerances: outputs are rounded once from 32 bits, half a step of the type (eps / 2 relative to the
value). The 32-bit rotation adds the angle's and the products' errors: |x| times about 1.2e-6 (an
angle good to 2 pi 2^-25 = 1.9e-7, cos and sin to 2 ulp, two products and a sum to 3 * 2^-24), x0 and
x1 of up to 5 standard deviations, and 2 x 5 x 6e-7 = 6e-6 bounds it. The norms' 32-bit sums of up to
512 terms and the reciprocal root are good to about 512 * 2^-24 / 2 = 1.5e-5 relative in the worst
case, taken as 2e-5."""
import math

import pytest
import torch

import dsa_triton_ascend_amd as dsa

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def freqs(pairs, base=10000.0, dev="cuda"):
    return (1.0 / base ** (torch.arange(pairs, dtype=torch.float32) / pairs)).to(dev)


def turned(x, positions, freq, sections, start, inter, back=False):
    """64-bit rotation of x [..., N, W] on the CPU."""
    x, p, f = x.detach().cpu().double().clone(), positions.cpu().double(), freq.cpu().double()
    if sections:
        axis = sum(([a] * n for a, n in enumerate(sections)), [])
        ang = torch.stack([p[a] for a in axis], -1) * f
    else:
        ang = p[..., None] * f
    ang = (-ang if back else ang).unsqueeze(-2)
    c, s, r = ang.cos(), ang.sin(), 2 * f.numel()
    part = x[..., start:start + r].clone()
    a, b = (part[..., 0::2], part[..., 1::2]) if inter else (part[..., :r // 2], part[..., r // 2:])
    a, b = a * c - b * s, a * s + b * c
    x[..., start:start + r] = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return x


def near(got, want, abs_tol, rel=0.0):
    # below the smallest normal number the step no longer shrinks with the value: half of it,
    # smallest_normal * eps / 2 (fp16: 2^-14 * 2^-10 / 2 = 2^-25), is the rounding's bound there
    fi = torch.finfo(got.dtype)
    d = (got.cpu().double() - want).abs()
    lim = (fi.eps / 2 + rel) * want.abs() + abs_tol + fi.smallest_normal * fi.eps / 2
    assert torch.isfinite(got).all()
    assert bool((d <= lim).all()), f"off by {(d - lim).max():.3e} over the bound"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("lead,heads,width,start,rdim,sections", [
    ((1, 1), 1, 64, 0, 64, None), ((3, 5), 128, 64, 0, 64, None), ((257,), 2, 128, 0, 64, None),
    ((2, 3), 3, 192, 128, 64, None), ((77,), 16, 128, 0, 128, (16, 24, 24)), ((2, 9), 5, 96, 32, 48, (8, 0, 15, 1)),
    ((7,), 1, 576, 512, 64, (30, 2)), ((3, 1), 7, 10, 3, 6, None), ((5,), 130, 2, 0, 2, (1,)), ((33,), 65, 160, 8, 80, None),
    ((4100,), 80, 64, 0, 64, None)])
def test_rotary(dtype, inter, lead, heads, width, start, rdim, sections):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(*lead, heads, width, generator=g).to(dtype).cuda()
    axes = (len(sections),) if sections else ()
    pos = torch.randint(0, 130000, axes + lead, generator=g).cuda()
    if width % 2 == 0 and heads % 2:
        pos = pos.int()
    f = freqs(rdim // 2)
    layout = "BSND" if len(lead) == 2 else "TND"
    kw = dict(sections=sections, rotary_start=start, interleaved=inter, layout=layout)
    for fn, back in ((dsa.rotary_embedding, False), (dsa.rotary_embedding_grad, True)):
        y = fn(x, pos, f, **kw)
        assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
        near(y, turned(x, pos, f, sections, start, inter, back), 6e-6)
        rest = [i for i in range(width) if not start <= i < start + rdim]
        assert torch.equal(y[..., rest], x[..., rest])


@pytest.mark.parametrize("inter", [True, False])
def test_rotary_far_positions(inter):
    """Positions past 2^31: an int64 position times its frequency keeps its fraction of a turn (the
    64-bit product is off by 2^-52 of 2^33 / 2 pi turns, 1e-6 of a radian)."""
    x = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(1)).cuda()
    pos = torch.tensor([2 ** 33 + 12345, 2 ** 31, -7, 0]).cuda()
    f = freqs(32)
    y = dsa.rotary_embedding(x, pos, f, interleaved=inter, layout="TND")
    near(y, turned(x, pos, f, None, 0, inter), 3e-5)
    assert torch.equal(y[3], x[3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["slice", "odd", "heads", "batch", "last", "expand", "broadcast", "one batch"])
def test_rotary_strides(dtype, how):
    g = torch.Generator().manual_seed(6)
    B, S, N, W = 3, 4, 6, 64
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    x = {"slice": lambda: r(B, S, N, 192)[..., 128:], "odd": lambda: r(B, S, N, W + 3)[..., 1:W + 1],
         "heads": lambda: r(B, S, W * N).view(B, S, N, W).transpose(1, 2).contiguous().transpose(1, 2),
         "batch": lambda: r(S, B, N, W).transpose(0, 1), "last": lambda: r(B, S, W, N).transpose(2, 3),
         "expand": lambda: r(B, S, 1, W).expand(B, S, N, W), "broadcast": lambda: r(1, S, 1, W).expand(B, S, N, W),
         "one batch": lambda: r(7, S, N, W)[3::4]}[how]()
    B = x.shape[0]
    pos = torch.randint(0, 9000, (B, S), generator=g).cuda()
    f = freqs(32)
    for inter in (True, False):
        near(dsa.rotary_embedding(x, pos, f, interleaved=inter), turned(x, pos, f, None, 0, inter), 6e-6)


def test_rotary_gradient_against_differences():
    """<d, rotate(x + h v) - rotate(x - h v)> / 2h is <rotary_embedding_grad(d), v>: exact for a linear
    map but for 32-bit roundings (3e-7 of the terms, 2000 of them with random signs over h = 1/2)."""
    g = torch.Generator().manual_seed(7)
    x, v, d = (torch.randn(11, 3, 128, generator=g).cuda() for _ in range(3))
    pos = torch.randint(0, 5000, (3, 11), generator=g).cuda()
    kw = dict(sections=(10, 10, 12), rotary_start=32, interleaved=False, layout="TND")
    f, h = freqs(32), 0.5
    up, down = (dsa.rotary_embedding(x + s * h * v, pos, f, **kw) for s in (1, -1))
    want = ((up.double() - down.double()) / (2 * h) * d.double()).sum()
    got = (dsa.rotary_embedding_grad(d, pos, f, **kw).double() * v.double()).sum()
    assert abs(float(want - got)) < 2e-4
    back = dsa.rotary_embedding_grad(dsa.rotary_embedding(x, pos, f, **kw), pos, f, **kw)
    assert float((back - x).abs().max()) < 1e-5


def test_rotary_empty_module_and_stream():
    f = freqs(32)
    assert dsa.rotary_embedding(torch.empty(0, 4, 64, device="cuda"), torch.empty(0, dtype=torch.long, device="cuda"), f,
                                layout="TND").shape == (0, 4, 64)
    x = torch.randn(2, 3, 4, 64, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(6, device="cuda").view(2, 3)
    m = dsa.RotaryEmbedding(f.cpu(), interleaved=False).cuda()
    want = dsa.rotary_embedding(x, pos, f, interleaved=False)
    assert torch.equal(m(x, pos), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = dsa.rotary_embedding(x, pos, f, interleaved=False)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dsa.rotary_embedding_grad(x, pos, f, interleaved=False)
    for k in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, dsa.rotary_embedding_grad(x, pos, f, interleaved=False)), k


# ------------------------------------------------------------------ appends
def places(table, tokens, kv, page, blocks):
    """(row of the packed new tokens, position, cache row) of each token that has a place."""
    got, at = [], 0
    for b, (t, k) in enumerate(zip(tokens, kv)):
        for s in range(t):
            p = k - t + s
            if p >= 0 and p // page < table.shape[1]:
                blk = int(table[b, p // page])
                if 0 <= blk < blocks:
                    got.append((at + s, p, blk * page + p % page))
        at += t
    return [torch.tensor(v, dtype=torch.long) for v in zip(*got)] if got else [torch.zeros(0, dtype=torch.long)] * 3


def block_table(kv, page, g, width=None):
    need = [-(-k // page) for k in kv]
    order = torch.randperm(sum(need) + 3, generator=g).int()
    table = torch.full((len(kv), width or max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


TOKENS = [([1], [1]), ([1, 1, 1], [7, 400, 33]), ([3, 0, 9, 2], [3, 5, 60, 2]), ([70, 1, 130], [70, 90, 131]),
          ([2, 4], [1, 4])]   # the last: a sequence shorter than its new tokens (the first token has no place)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,kv", TOKENS)
@pytest.mark.parametrize("d,page,norm,inter", [(512, 64, "io", True), (256, 48, "fp32", False), (128, 1, None, True)])
def test_latent_append(dtype, tokens, kv, d, page, norm, inter):
    g = torch.Generator().manual_seed(8)
    T = sum(tokens)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    table, blocks = block_table(kv, page, g)
    if T > 100:
        table[0, 0] = -1               # a missing page: its tokens are not stored
        table[2, 1] = blocks           # one past the cache: neither
    latent, rope = r(T + 5, 1, d) * 3, r(T + 5, 1, 64)      # 5 rows behind the last sequence
    cache, rcache = r(blocks, page, 1, d), r(blocks, page, 1, 64)
    w = None if norm is None else (1 + 0.2 * torch.randn(d, generator=g)).to(dtype if norm == "io" else torch.float32)
    f = freqs(32, dev="cpu")
    rows, pos, slots = places(table, tokens, kv, page, blocks)
    want, rwant = cache.double().view(-1, d), rcache.double().view(-1, 64)
    x = latent.double()[:, 0]
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
    want[slots] = x[rows]
    rwant[slots] = turned(rope[rows], pos, f, None, 0, inter)[:, 0]
    cu = torch.tensor(tokens).cumsum(0).tolist()
    c, rc = cache.cuda(), rcache.cuda()
    out = dsa.latent_cache_append(latent.cuda(), rope.cuda(), c, rc, table.cuda(), f.cuda(), kv, cu,
                                  norm_weight=None if w is None else w.cuda(), norm_eps=1e-5, interleaved=inter,
                                  layout="TND")
    assert out[0] is c and out[1] is rc
    near(c.view(-1, d), want, 0, 2e-5)
    near(rc.view(-1, 64), rwant, 6e-6)
    rest = torch.ones(blocks * page, dtype=torch.bool)
    rest[slots] = False                # every other row as it was
    assert torch.equal(c.cpu().view(-1, d)[rest], cache.view(-1, d)[rest])
    assert torch.equal(rc.cpu().view(-1, 64)[rest], rcache.view(-1, 64)[rest])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,kv", TOKENS)
@pytest.mark.parametrize("n2,w,start,rdim,inter,norm,bias", [
    (1, 128, 0, 64, False, True, True), (2, 64, 0, 64, True, True, False), (3, 96, 8, 48, False, True, True),
    (1, 256, 64, 128, False, False, False), (5, 512, 0, 512, False, True, True), (33, 64, 32, 32, True, True, True)])
def test_index_append(dtype, tokens, kv, n2, w, start, rdim, inter, norm, bias):
    g = torch.Generator().manual_seed(9)
    T, page = sum(tokens), 16
    table, blocks = block_table(kv, page, g, width=30)
    key = (torch.randn(T, n2, w, generator=g) * 2 + 0.5).to(dtype)
    cache = torch.randn(blocks, page, n2, w, generator=g).to(dtype)
    wt = 1 + 0.2 * torch.randn(w, generator=g) if norm else None
    bs = 0.3 * torch.randn(w, generator=g) if bias else None
    f = freqs(rdim // 2, dev="cpu")
    rows, pos, slots = places(table, tokens, kv, page, blocks)
    x = key.double()
    if norm:
        x = x - x.mean(-1, keepdim=True)
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * wt.double()
        x = x + bs.double() if bias else x
    axes = (3, 2, rdim // 2 - 5)
    ppos = torch.randint(0, 3000, (3, T), generator=g, dtype=torch.int32)
    for explicit in (False, True):
        y = turned(x[rows], ppos[:, rows] if explicit else pos, f, axes if explicit else None, start, inter)
        want = cache.double().view(-1, n2, w)
        want[slots] = y
        c = cache.cuda()
        cu = torch.tensor(tokens).cumsum(0).tolist()
        out = dsa.index_cache_append(key.cuda(), c, table.cuda(), f.cuda(), kv, cu,
                                     positions=ppos.cuda() if explicit else None, sections=axes if explicit else None,
                                     norm_weight=None if wt is None else wt.cuda(),
                                     norm_bias=None if bs is None else bs.cuda(), rotary_start=start, interleaved=inter,
                                     layout="TND")
        assert out is c
        # values before the rotation up to 5 x 1.6, so the absolute part grows with them
        near(c.view(-1, n2, w), want, 2e-4 if not norm else 1e-4, 2e-5)
        rest = torch.ones(blocks * page, dtype=torch.bool)
        rest[slots] = False
        assert torch.equal(c.cpu().view(-1, n2, w)[rest], cache.view(-1, n2, w)[rest])


def test_append_strides_and_constant_rows():
    """Slices of a fused projection (rows of 512 + 64 + 128, one element in), BSND with fewer tokens
    than S, and vectors of one value (variance 0: the norm's eps alone keeps it finite)."""
    g = torch.Generator().manual_seed(10)
    B, S, page = 2, 5, 16
    for off in (0, 1):
        buf = torch.randn(B, S, 1, 712, generator=g).bfloat16()
        buf[0, 1] = 0
        fused = buf.cuda()[..., off:]
        latent, rope, key = fused[..., :512], fused[..., 512:576], fused[..., 576:704]
        table = torch.randperm(6, generator=g).int().view(2, 3).cuda()
        kv, nq = [20, 48], [5, 2]
        f = freqs(32)
        c, rc, ic = (torch.zeros(6, page, 1, n, dtype=torch.bfloat16, device="cuda") for n in (512, 64, 128))
        one = torch.ones(512, device="cuda")
        dsa.latent_cache_append(latent, rope, c, rc, table, f, kv, nq, norm_weight=one)
        dsa.index_cache_append(key, ic, table, f, kv, nq, norm_weight=one[:128])
        h = buf.double()[..., off:]
        for b in range(B):
            for s in range(S):
                p = kv[b] - nq[b] + s
                at = (int(table[b, p // page]), p % page) if s < nq[b] else None
                if at is None:
                    continue
                x = h[b, s, 0, :512]
                near(c[at][0], x / (x.square().mean() + 1e-6).sqrt(), 1e-30, 2e-5)
                near(rc[at][0], turned(h[b, s, :, 512:576], torch.tensor(p), f, None, 0, True)[0], 6e-6)
                y = h[b, s, 0, 576:704]
                y = (y - y.mean()) / ((y - y.mean()).square().mean() + 1e-6).sqrt()
                near(ic[at][0], turned(y[None], torch.tensor(p), f, None, 0, False)[0], 1e-4, 2e-5)
        assert int((c.abs().sum(-1) > 0).sum()) == sum(nq) - 1   # the zero vector stays zero


@pytest.mark.parametrize("batch", [17, 18, 19, 40])
def test_append_lengths_as_arguments_and_uploaded(batch):
    """One-shot calls up to 18 sequences take their lengths along, longer ones and plans upload them: the same
    caches from both, uneven packed sequences with empty ones and rows behind the last among them."""
    g = torch.Generator().manual_seed(14)
    tokens = torch.randint(0, 5, (batch,), generator=g).tolist()
    kv = [t + int(torch.randint(0, 40, (1,), generator=g)) for t in tokens]
    table, blocks = block_table(kv, 8, g)
    T, cu = sum(tokens) + 2, torch.tensor(tokens).cumsum(0).tolist()
    x, r = torch.randn(T, 1, 256, generator=g).half().cuda(), torch.randn(T, 1, 64, generator=g).half().cuda()
    key = torch.randn(T, 2, 64, generator=g).half().cuda()
    f, got = freqs(32), []
    for plan in (False, True):
        c, rc, ic = (torch.zeros(blocks, 8, n, w, dtype=torch.half, device="cuda") for n, w in ((1, 256), (1, 64), (2, 64)))
        if plan:
            dsa.LatentAppendPlan(x, r, c, rc, table.cuda(), f, kv, cu, layout="TND").run()
            dsa.IndexAppendPlan(key, ic, table.cuda(), f, kv, cu, layout="TND").run()
        else:
            dsa.latent_cache_append(x, r, c, rc, table.cuda(), f, kv, cu, layout="TND")
            dsa.index_cache_append(key, ic, table.cuda(), f, kv, cu, layout="TND")
        got.append((c, rc, ic))
    rows, pos, slots = places(table, tokens, kv, 8, blocks)
    want = torch.zeros(blocks * 8, 256, dtype=torch.half)
    want[slots] = x.cpu()[rows, 0]
    assert torch.equal(got[0][0].cpu().view(-1, 256), want)
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_append_broadcast_tokens():
    """The same new tokens for every sequence (a batch stride of 0), and a batch of one cut from more."""
    x, r = torch.randn(1, 3, 1, 128).half().cuda(), torch.randn(1, 3, 1, 64).half().cuda()
    table = torch.arange(8).int().view(4, 2).cuda()
    for tokens, rows in ((x.expand(4, 3, 1, 128), 4), (torch.cat([x * 0, x, x * 0])[1::2], 1)):
        c, rc = (torch.zeros(8, 4, 1, w, dtype=torch.half, device="cuda") for w in (128, 64))
        dsa.latent_cache_append(tokens, r.expand(rows, 3, 1, 64), c, rc, table[:rows], freqs(32), [5] * rows)
        for b in range(rows):
            got = c[table[b].long()].reshape(8, 128)
            assert torch.equal(got[2:5], x[0, :, 0]) and not got[:2].any() and not got[5:].any()


def test_append_far_cache_rows():
    """Cache rows past 2^31 bytes (and elements): block 70000 of 64 tokens of 512."""
    cache = torch.zeros(70001, 64, 1, 512, dtype=torch.bfloat16, device="cuda")
    rcache = torch.zeros(70001, 64, 1, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(1, 1, 1, 512, device="cuda").bfloat16()
    r = torch.randn(1, 1, 1, 64, device="cuda").bfloat16()
    dsa.latent_cache_append(x, r, cache, rcache, torch.tensor([[70000]], device="cuda"), freqs(32), [64])
    assert torch.equal(cache[70000, 63, 0], x[0, 0, 0]) and int((cache != 0).any(-1).sum()) == 1
    assert int((rcache != 0).any(-1).sum()) == 1


def test_append_plan_replays_with_new_lengths():
    """A captured run() reads act_k and the block table on the device: the next token's place after each
    step, and a padded sequence (length 0: no place) in the batch."""
    g = torch.Generator().manual_seed(11)
    B, page = 3, 16
    table = torch.randperm(12, generator=g).int().view(B, 4).cuda()
    x = torch.zeros(B, 1, 1, 512, dtype=torch.bfloat16, device="cuda")
    r = torch.zeros(B, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    c, rc = (torch.zeros(12, page, 1, n, dtype=torch.bfloat16, device="cuda") for n in (512, 64))
    build = torch.cuda.Stream()
    with torch.cuda.stream(build):
        plan = dsa.LatentAppendPlan(x, r, c, rc, table, freqs(32), [15, 0, 40])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    want = torch.zeros(12, page, 512, dtype=torch.bfloat16)
    for step in range(4):
        lens = [15 + step, 0, 40 + step]
        plan.act_k[:B].copy_(torch.tensor(lens, dtype=torch.int32))
        x.copy_(torch.randn(B, 1, 1, 512, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        for b, k in enumerate(lens):
            if k:
                want[int(table[b, (k - 1) // page]), (k - 1) % page] = x[b, 0, 0].cpu()
        assert torch.equal(c[:, :, 0].cpu(), want), step


def test_append_plan_is_in_place_when_built(monkeypatch):
    """A plan's own copies (here of norm weights with a stride) are made before the wait in its constructor:
    a run on another stream right after it reads them, however busy the building stream is then."""
    from dsa_triton_ascend_amd import _host

    upload = _host.upload

    def upload_then_busy(*args, **kw):
        lengths = upload(*args, **kw)
        torch.cuda._sleep(100_000_000)
        return lengths

    g = torch.Generator().manual_seed(21)
    table = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2)
    x = torch.randn(1, 3, 1, 512, generator=g).bfloat16().cuda()
    k = torch.randn(1, 3, 1, 128, generator=g).bfloat16().cuda()
    r = torch.zeros(1, 3, 1, 64, dtype=torch.bfloat16, device="cuda")
    w = (1 + torch.rand(512, 2, generator=g)).cuda()
    freq = freqs(32)
    caches = lambda width: torch.zeros(2, 16, 1, width, dtype=torch.bfloat16, device="cuda")
    want = dsa.latent_cache_append(x, r, caches(512), caches(64), table, freq, [3], norm_weight=w[:, 0].contiguous())[0].cpu()
    want_k = dsa.index_cache_append(k, caches(128), table, freq, [3], norm_weight=w[:128, 0].contiguous(),
                                    norm_bias=w[:128, 1].contiguous()).cpu()
    c, rc, ck = caches(512), caches(64), caches(128)
    torch.cuda.synchronize()
    monkeypatch.setattr(_host, "upload", upload_then_busy)
    build, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(build):
        plan = dsa.LatentAppendPlan(x, r, c, rc, table, freq, [3], norm_weight=w[:, 0])
        with torch.cuda.stream(other):
            plan.run()
        other.synchronize()
        keys = dsa.IndexAppendPlan(k, ck, table, freq, [3], norm_weight=w[:128, 0], norm_bias=w[:128, 1])
        with torch.cuda.stream(other):
            keys.run()
        other.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(c.cpu(), want) and torch.equal(ck.cpu(), want_k)


@pytest.mark.parametrize("sections", [None, (8, 12, 12)])
def test_prefill_rotates(sections):
    """dsa_prefill with inverse frequencies: the bits of rotating first and calling it as before, from a
    plan run twice with new contents too."""
    g = torch.Generator().manual_seed(13)
    lens, dt = [70, 33, 120], torch.bfloat16
    T, cu = sum(lens), torch.tensor(lens).cumsum(0).tolist()
    r = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    iq, ik, iw = r(T, 32, 128), r(T, 1, 128), torch.randn(T, 32, generator=g).cuda()
    q, k, qr, kr = r(T, 16, 512), r(T, 1, 512), r(T, 16, 64), r(T, 1, 64)
    f = freqs(32)
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    if sections:
        pos = torch.randint(0, 500, (3, T), generator=g).cuda()
    kw = dict(sparse_count=32, scale_value=0.04, return_softmax_lse=True)
    plan = dsa.PrefillPlan(iq, ik, iw, q, k, qr, kr, cu, inv_freq=f, positions=pos if sections else None, sections=sections, **kw)
    for step in range(2):
        rot = [dsa.rotary_embedding(x, pos, f, sections=sections, layout="TND") for x in (qr, kr)]
        want = dsa.dsa_prefill(iq, ik, iw, q, k, *rot, cu, **kw)
        got = plan.run()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), step
        assert torch.equal(got[1], dsa.dsa_prefill(iq, ik, iw, q, k, qr, kr, cu, inv_freq=f, positions=pos, sections=sections, **kw)[1])
        qr.copy_(r(T, 16, 64))
    if not sections:   # captured whole, positions and all
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = dsa.dsa_prefill(iq, ik, iw, q, k, qr, kr, cu, inv_freq=f, **kw)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, plan.run()))
            torch.cuda.synchronize()


def test_prefill_then_sparse_attention():
    """The operators as a layer uses them: queries rotated, keys of two prompts appended to the paged
    caches, indexer and sparse attention over them; the same as both on contiguous keys rotated and
    normed beforehand by the 64-bit forms (indices by the indexer's own rule on the cache's contents)."""
    g = torch.Generator().manual_seed(12)
    B, S, N, page = 2, 80, 16, 16
    dt, dev = torch.bfloat16, "cuda"
    rnd = lambda *s: torch.randn(*s, generator=g).to(dt)
    latent, rope, ikey = rnd(B, S, 1, 512), rnd(B, S, 1, 64), rnd(B, S, 1, 128)
    q, qr, iq, iw = rnd(B, S, N, 512), rnd(B, S, N, 64), rnd(B, S, 32, 128), torch.randn(B, S, 32, generator=g)
    table = torch.randperm(12, generator=g).int()[:10].view(B, 5)
    f = freqs(32)
    pos = torch.arange(S).expand(B, S)
    c, rc, ic = (torch.zeros(12, page, 1, n, dtype=dt, device=dev) for n in (512, 64, 128))
    w = (1 + 0.1 * torch.randn(512, generator=g)).to(dt)
    dsa.latent_cache_append(latent.to(dev), rope.to(dev), c, rc, table.to(dev), f, [S] * B, norm_weight=w.to(dev))
    dsa.index_cache_append(ikey.to(dev), ic, table.to(dev), f, [S] * B)
    qrot = dsa.rotary_embedding(qr.to(dev), pos.to(dev), f)
    irot = dsa.rotary_embedding(iq.to(dev), pos.to(dev), f, interleaved=False)
    idx, _ = dsa.lightning_indexer(irot, ic, iw.to(dev), actual_seq_lengths_key=[S] * B, block_table=table.to(dev),
                                   layout_key="PA_BSND", sparse_count=32)
    out, _, _ = dsa.sparse_flash_attention(q.to(dev), c, c, idx, 576 ** -0.5, table.to(dev), None, [S] * B, qrot, rc,
                                           layout_kv="PA_BSND", sparse_mode=3)
    flat = lambda t, n: t.cpu()[table.long()].reshape(B, S, 1, n)
    k, kr, ki = flat(c, 512), flat(rc, 64), flat(ic, 128)
    x = latent.double()
    near(k, x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double(), 0, 2e-5)
    near(kr, turned(rope, pos, f, None, 0, True), 6e-6)
    near(ki, turned(ikey, pos, f, None, 0, False), 6e-6)
    idx2, _ = dsa.lightning_indexer(irot, ki.to(dev), iw.to(dev), sparse_count=32)
    assert torch.equal(idx, idx2)
    out2, _, _ = dsa.sparse_flash_attention(q.to(dev), k.to(dev), k.to(dev), idx, 576 ** -0.5, query_rope=qrot,
                                            key_rope=kr.to(dev), sparse_mode=3)
    assert float((out.float() - out2.float()).abs().max()) <= 2 ** -6 * float(out2.float().abs().max())


@pytest.mark.parametrize("lengths,tail", [([5], 0), ([0, 3, 0, 0, 300, 1], 9), ([257] * 70 + [0], 0), ([0], 3), ([], 4)])
def test_row_positions(lengths, tail):
    from dsa_triton_ascend_amd.rotary import _row_positions
    rows = sum(lengths) + tail
    want = [p for n in lengths for p in range(n)] + [0] * tail
    assert _row_positions(lengths, rows, torch.device("cuda")).tolist() == want


def test_prefill_makes_its_positions_without_waiting():
    """A one-shot dsa_prefill that rotates only queues work: the host does not wait for what runs before it."""
    g = torch.Generator().manual_seed(15)
    lens, dt = [300, 0, 212], torch.bfloat16
    T, cu = sum(lens), torch.tensor(lens).cumsum(0).tolist()
    r = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    args = (r(T, 32, 128), r(T, 1, 128), torch.randn(T, 32, generator=g).cuda(), r(T, 16, 512), r(T, 1, 512), r(T, 16, 64),
            r(T, 1, 64), cu)
    kw = dict(sparse_count=64, scale_value=0.04)
    f = freqs(32)
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    want = dsa.dsa_prefill(*args, inv_freq=f, positions=pos, **kw)
    dsa.dsa_prefill(*args, inv_freq=f, **kw)   # the allocator has its memory
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    before = torch.cuda.Event()
    before.record()
    got = dsa.dsa_prefill(*args, inv_freq=f, **kw)
    assert not before.query()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rotary_of_more_rows_than_one_grid_dimension():
    """2^24 work-groups and more (rows of one each): 2^32 threads would not fit a launch's x."""
    rows = 2 ** 24 + 13
    x = torch.randn(1, 130, 2, generator=torch.Generator().manual_seed(22)).bfloat16().cuda().expand(rows, 130, 2)
    pos = (torch.arange(rows, dtype=torch.int32) % 7).cuda()
    y = dsa.rotary_embedding(x, pos, freqs(1), layout="TND")
    near(y[:7], turned(x[:7], pos[:7], freqs(1), None, 0, True), 6e-6)
    assert rows % 7 == 0 and bool((y.view(-1, 7, 130, 2) == y[:7]).all())


def test_append_of_more_tokens_than_one_grid_dimension():
    """2^24 work-groups of eight tokens and more; all but the first and the last tokens have no block."""
    T, page = 2 ** 27 + 9, 2 ** 20
    key = torch.randn(1, 1, 64, generator=torch.Generator().manual_seed(23)).half().cuda().expand(T, 1, 64)
    cache = torch.zeros(2, page, 1, 64, dtype=torch.half, device="cuda")
    table = torch.full((1, 129), -1, dtype=torch.int32)
    table[0, 0], table[0, 128] = 1, 0
    f = freqs(32)
    dsa.index_cache_append(key, cache, table.cuda(), f, [T], [T], layout="TND")
    for block, pos in ((1, torch.arange(page)), (0, torch.arange(2 ** 27, T))):
        # (the 64-bit angle of a position below 2^27 is good to 2^27 2^-52 = 3e-8: inside the bound)
        near(cache[block, :len(pos)], turned(key[:len(pos)], pos, f, None, 0, False), 6e-6)
        assert not cache[block, len(pos):].any()


@pytest.mark.parametrize("heads,width,start", [(128, 64, 0), (131, 72, 8)])
def test_rotary_of_many_units(heads, width, start):
    """2^24 units of 16 bytes and more (four a thread), whole rows of work-groups and ragged ones, both directions."""
    rows = 2 ** 24 // (heads * (width // 8)) + 3
    x = torch.randn(rows, heads, width, device="cuda", generator=torch.Generator("cuda").manual_seed(24)).bfloat16()
    pos, f = torch.arange(rows).cuda() * 7, freqs(32)
    pick = torch.cat([torch.arange(40), torch.randint(0, rows, (200,), generator=torch.Generator().manual_seed(25)),
                      torch.arange(rows - 40, rows)])
    for fn, back in ((dsa.rotary_embedding, False), (dsa.rotary_embedding_grad, True)):
        y = fn(x, pos, f, rotary_start=start, layout="TND")
        near(y[pick.cuda()], turned(x[pick.cuda()], pos[pick.cuda()], f, None, start, True, back), 6e-6)
        assert torch.equal(y[..., :start], x[..., :start]) and torch.equal(y[..., start + 64:], x[..., start + 64:])
        few = torch.cat([fn(p, q, f, rotary_start=start, layout="TND") for p, q in zip(x.split(2000), pos.split(2000))])
        # the small calls' roundings may differ: at most a step of the value, and 32-bit errors of both
        assert bool(((y.float() - few.float()).abs() <= 2.0 ** -7 * few.float().abs() + 1.2e-5).all())


def test_prefill_plan_that_rotates_runs_on_another_stream():
    """A kept PrefillPlan's positions are in place when its constructor returns, however busy the stream it was built on."""
    g = torch.Generator().manual_seed(26)
    lens, dt = [90, 0, 40], torch.bfloat16
    T, cu = sum(lens) + 6, torch.tensor(lens).cumsum(0).tolist()   # six rows behind the last sequence
    r = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    args = (r(T, 32, 128), r(T, 1, 128), torch.randn(T, 32, generator=g).cuda(), r(T, 16, 512), r(T, 1, 512), r(T, 16, 64),
            r(T, 1, 64), cu)
    kw = dict(sparse_count=32, scale_value=0.04, inv_freq=freqs(32))
    pos = torch.cat([torch.arange(n) for n in lens] + [torch.zeros(6, dtype=torch.long)]).cuda()
    want = [o.clone() for o in dsa.PrefillPlan(*args, positions=pos, **kw).run()]
    torch.cuda.synchronize()
    build, use = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(build):
        torch.cuda._sleep(40_000_000)
        plan = dsa.PrefillPlan(*args, **kw)
    with torch.cuda.stream(use):
        got = plan.run()
    torch.cuda.synchronize()
    n = sum(lens)
    assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1][:n], want[1][:n])
