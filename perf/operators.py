"""Rotary positions, writing the paged caches, and attention over a shared prefix, as measured cases.

``listed()`` holds the fixed cases, ``draw(rng)`` gives further ones of the same ranges. ``prepare``
makes what a program has in hand before the call, ``run`` is one pass: with ``own`` the package's
operators, else the same operators written out in elementary torch. ``exact`` computes a case's
outputs in 64 bits from the definitions, apart from both.

Kinds of case:
  rotate   ``rotary_embedding`` on the rotary part of a model's queries (or on an indexer's queries, of
           which the first dimensions turn), ``rotary_embedding_grad`` on their gradients, or both
  latent   one layer's new latent and rotary keys into the paged caches that the attention reads:
           norm, rotation and the store
  index    one layer's new indexer keys into the indexer's paged cache
  attend   attention over paged latents for a batch whose sequences begin with the same tokens
"""
import math
import random

import torch

own = False

ROPE = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _numbers(text):
    return [int(v) for v in text.split(",") if v]


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _spread(n, low, high, seed):
    """n lengths between low and high, even over the range, in no order."""
    r = random.Random(seed)
    got = [round(low + (high - low) * (i + 0.5) / n) for i in range(n)]
    r.shuffle(got)
    return got


def listed():
    return [
        # the queries of one decode step, 16 sequences, all 128 heads: launch and host time count
        dict(name="rotate_decode", kind="rotate", dtype="bf16", tokens="1," * 15 + "1", packed=False, heads=128,
             width=64, rotary=64, start=0, interleaved=True, sections="", ways="forward", far=30000),
        # the queries of a packed prefill of ragged prompts, far into the context
        dict(name="rotate_prompt", kind="rotate", dtype="bf16", tokens="1024,2000,5168", packed=True, heads=128,
             width=64, rotary=64, start=0, interleaved=True, sections="", ways="forward", far=100000),
        # training: gradient of the indexer's queries, half of whose dimensions turn, pairs half a width apart
        dict(name="rotate_index_grad", kind="rotate", dtype="bf16", tokens="4093", packed=False, heads=64,
             width=128, rotary=64, start=0, interleaved=False, sections="", ways="grad", far=0),
        # video tokens: time, height and width on axes of their own, 32-bit tensors, forward and gradient
        dict(name="rotate_video", kind="rotate", dtype="fp32", tokens="2501,2502", packed=True, heads=16,
             width=128, rotary=128, start=0, interleaved=False, sections="16,24,24", ways="both", far=4000),
        # one decode step's keys of one layer, 64 sequences
        dict(name="latent_decode", kind="latent", dtype="bf16", tokens=_text([1] * 64), packed=False, dim=512,
             kv=_text(_spread(64, 200, 2400, 1)), page=64, norm=True, interleaved=True),
        # the keys of four packed prompts, all of it new
        dict(name="latent_prompts", kind="latent", dtype="bf16", tokens="1024,3000,6000,8192", packed=True, dim=512,
             kv="1024,3000,6000,8192", page=128, norm=True, interleaved=True),
        # the indexer's keys of a speculative step: three tokens a sequence
        dict(name="index_decode", kind="index", dtype="bf16", tokens=_text([3] * 48), packed=False, heads=1, width=128,
             rotary=64, kv=_text(_spread(48, 64, 1800, 2)), page=64, norm=True, interleaved=False),
        # the indexer's keys of chunks of long prompts, odd sizes and pages, two key heads
        dict(name="index_prompts", kind="index", dtype="fp16", tokens="777,4099,2050", packed=True, heads=2, width=128,
             rotary=64, kv="777,9001,2600", page=48, norm=True, interleaved=False),
        # the smallest attention call: a few sequences after a short system prompt
        dict(name="attend_small", kind="attend", dtype="bf16", heads=16, dim=512, prefix=304, tokens="1,1,1,1",
             packed=False, kv="305,311,340,327", page=16, lse=False),
        # a decode step with 16 heads on this GPU (eight-way tensor parallel): 64 sequences after 8K shared tokens
        dict(name="attend_decode_h16", kind="attend", dtype="bf16", heads=16, dim=512, prefix=8192,
             tokens=_text([1] * 64), packed=False, kv=_text(_spread(64, 8193, 9700, 3)), page=64, lse=False),
        # a decode step with all 128 heads: 32 sequences after 16K shared tokens, odd lengths
        dict(name="attend_decode_h128", kind="attend", dtype="bf16", heads=128, dim=512, prefix=16384,
             tokens=_text([1] * 32), packed=False, kv=_text(_spread(32, 16500, 20001, 4)), page=128, lse=False),
        # questions of some hundred tokens about one document of 2K tokens, packed, statistics wanted
        dict(name="attend_prompts", kind="attend", dtype="fp16", heads=64, dim=512, prefix=2048,
             tokens="97,301,500,412,655", packed=True, kv="2145,2349,2548,2460,2703", page=64, lse=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _parts(rng, total, most):
    """`total` tokens as up to `most` sequences of uneven lengths."""
    n = min(rng.randint(1, most), total)
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    kind = rng.choice(["rotate", "latent", "index", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    c = dict(kind=kind, dtype=dtype)
    if kind == "rotate":
        heads, (width, rotary, start) = rng.choice([1, 8, 16, 64, 128]), rng.choice(
            [(64, 64, 0), (64, 64, 0), (128, 64, 0), (128, 128, 0), (192, 64, 128), (576, 64, 512)])
        total = _log(rng, 1, min(8192, 60_000_000 // (heads * width)))
        packed = rng.random() < 0.5
        c.update(dtype=rng.choice([dtype, "fp32"]), packed=packed, heads=heads, width=width, rotary=rotary, start=start,
                 tokens=_text(_parts(rng, total, 6) if packed else [total]),
                 interleaved=rng.random() < 0.5, sections=rng.choice(["", "", "axes"]),
                 ways=rng.choice(["forward", "grad", "both"]), far=rng.choice([0, 5000, 120000]))
        if c["sections"]:
            a = rng.randint(1, rotary // 4)
            b = rng.randint(1, rotary // 4 - 1) if rotary > 8 else 1
            c["sections"] = _text([a, b, rotary // 2 - a - b])
        return c
    if kind in ("latent", "index"):
        decode = rng.random() < 0.4
        if decode:
            n, s = _log(rng, 1, 128), rng.choice([1, 1, 2, 4])
            tokens = [s] * n
        else:
            tokens = _parts(rng, _log(rng, 20, 16000), 6)
        earlier = [rng.choice([0, rng.randint(0, 3000)]) for _ in tokens]
        c.update(tokens=_text(tokens), packed=not decode, kv=_text(t + e for t, e in zip(tokens, earlier)),
                 page=rng.choice([16, 48, 64, 128]), norm=rng.random() < 0.8, interleaved=rng.random() < 0.5)
        if kind == "latent":
            c.update(dim=rng.choice([512, 512, 256, 128]))
        else:
            c.update(heads=rng.choice([1, 1, 2]), width=rng.choice([128, 128, 64, 256]), rotary=64)
        return c
    heads, dim, page = rng.choice([1, 8, 16, 16, 32, 64, 128]), rng.choice([512, 512, 512, 256, 128]), rng.choice([16, 48, 64, 128])
    decode = rng.random() < 0.6
    if decode:
        n, s = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 4])
        tokens = [s] * n
    else:
        tokens = _parts(rng, _log(rng, 30, 2000), 6)
    most = 60_000_000 // max(1, sum(tokens) * heads)   # head rows times tokens, below the largest listed case's
    prefix = _log(rng, 32, max(64, min(16384, most // 2)))
    prefix = rng.choice([prefix, max(page, prefix // page * page)])
    more = _log(rng, 1, max(2, min(3000, most // 4)))
    c.update(heads=heads, dim=dim, prefix=prefix, tokens=_text(tokens), packed=not decode,
             kv=_text(prefix + t + rng.randint(0, more) for t in tokens), page=page, lse=rng.random() < 0.5)
    return c


# ------------------------------------------------------------------ inputs
class _Source:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(seed)
        self.r = random.Random(seed)

    def normal(self, shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=self.g, device=self.dev, dtype=torch.float32) * scale).to(dtype)

    def tables(self, lengths, page, spare=3):
        """A block table over a pool in random order, -1 behind each sequence's pages: (table, blocks)."""
        need = [-(-v // page) for v in lengths]
        pool = sum(need) + spare
        order = list(range(pool))
        self.r.shuffle(order)
        table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        return table, pool


def _frequencies(rotary, dev):
    """Inverse frequencies of the pairs, base 10000, in float32 as checkpoints' code makes them."""
    return 1.0 / (10000.0 ** (torch.arange(0, rotary, 2, device=dev, dtype=torch.float32) / rotary))


def _lead(case):
    """(shape before the heads, rows) of a query-like tensor: packed rows, or [batch, tokens]."""
    t = _numbers(case["tokens"])
    return (sum(t),) if case["packed"] else (len(t), t[0])


def _starts(lengths):
    out = [0]
    for v in lengths:
        out.append(out[-1] + v)
    return out


def _query_lengths(case):
    t = _numbers(case["tokens"])
    return _starts(t)[1:] if case["packed"] else None


def _inputs(case, seed):
    s, dt = _Source(seed), DTYPES[case["dtype"]]
    lead, tokens, kind = _lead(case), _numbers(case["tokens"]), case["kind"]
    if kind == "rotate":
        x = s.normal(lead + (case["heads"], case["width"]), dt)
        d = s.normal(lead + (case["heads"], case["width"]), dt) if case["ways"] != "forward" else None
        steps = torch.cat([torch.arange(t) + s.r.randint(0, case["far"]) for t in tokens])
        sections = _numbers(case["sections"])
        if sections:   # time, height, width of each token of a video, 12 x 20 patches a frame
            steps = torch.stack([steps // 240, steps // 20 % 12, steps % 20])
        positions = steps.reshape(((len(sections),) if sections else ()) + lead).to(torch.int64).to(s.dev)
        return dict(x=x, d=d, positions=positions, freq=_frequencies(case["rotary"], s.dev))
    kv = _numbers(case["kv"])
    if kind == "latent":
        table, pool = s.tables(kv, case["page"])
        return dict(latent=s.normal(lead + (1, case["dim"]), dt, 2.0), rope=s.normal(lead + (1, ROPE), dt),
                    cache=s.normal((pool, case["page"], 1, case["dim"]), dt),
                    rope_cache=s.normal((pool, case["page"], 1, ROPE), dt), table=table.to(s.dev),
                    weight=(1 + 0.1 * s.normal((case["dim"],), torch.float32)).to(dt) if case["norm"] else None,
                    freq=_frequencies(ROPE, s.dev))
    if kind == "index":
        table, pool = s.tables(kv, case["page"])
        w = case["width"]
        return dict(keys=s.normal(lead + (case["heads"], w), dt, 1.5) + 0.25,
                    cache=s.normal((pool, case["page"], case["heads"], w), dt), table=table.to(s.dev),
                    weight=1 + 0.1 * s.normal((w,), torch.float32) if case["norm"] else None,
                    bias=0.1 * s.normal((w,), torch.float32) if case["norm"] else None,
                    freq=_frequencies(case["rotary"], s.dev))
    # attend: the pages of the whole prefix are the same in every row of the table; where the prefix
    # ends inside a page, each sequence has its own copy of that page
    page, whole = case["page"], case["prefix"] // case["page"]
    table, pool = s.tables([v - whole * page for v in kv], page, spare=whole + 2)
    free = sorted(set(range(pool)) - set(table.flatten().tolist()))
    s.r.shuffle(free)
    shared = torch.tensor(free[:whole], dtype=torch.int32).expand(len(kv), whole)
    table = torch.cat([shared, table], 1).contiguous()
    cache = s.normal((pool, page, 1, case["dim"]), dt)
    rope_cache = s.normal((pool, page, 1, ROPE), dt)
    over = case["prefix"] - whole * page
    if over:
        first = int(table[0, whole])
        for b in range(1, len(kv)):
            for c in (cache, rope_cache):
                c[int(table[b, whole]), :over] = c[first, :over]
    return dict(query=s.normal(lead + (case["heads"], case["dim"]), dt),
                query_rope=s.normal(lead + (case["heads"], ROPE), dt), cache=cache, rope_cache=rope_cache,
                table=table.to(s.dev))


def _scale(case):
    return 1.0 / math.sqrt(case["dim"] + ROPE)


def _kv_lengths(case):
    """Lengths as the attention takes them beside packed or BSND queries and a paged cache: per sequence."""
    return _numbers(case["kv"])


def prepare(case, seed):
    i = _inputs(case, seed)
    state = dict(case=case, i=i)
    kind = case["kind"]
    if kind == "rotate":
        return state
    if own and not case["packed"]:   # a serving loop keeps the plan of its step
        import dsa_triton_ascend_amd as dsa
        if kind == "latent":
            state["plan"] = dsa.LatentAppendPlan(i["latent"], i["rope"], i["cache"], i["rope_cache"], i["table"], i["freq"],
                                                 _kv_lengths(case), norm_weight=i["weight"],
                                                 interleaved=case["interleaved"])
        elif kind == "index":
            state["plan"] = dsa.IndexAppendPlan(i["keys"], i["cache"], i["table"], i["freq"], _kv_lengths(case),
                                                norm_weight=i["weight"], norm_bias=i["bias"],
                                                interleaved=case["interleaved"])
        else:
            state["plan"] = dsa.SharedPrefixPlan(i["query"], i["cache"], i["cache"], i["table"], case["prefix"],
                                                 _scale(case), None, _kv_lengths(case), query_rope=i["query_rope"],
                                                 key_rope=i["rope_cache"], return_softmax_lse=case["lse"])
    return state


def run(state):
    case, i = state["case"], state["i"]
    if not own:
        return _PLAIN[case["kind"]](case, i)
    import dsa_triton_ascend_amd as dsa
    kind = case["kind"]
    if kind == "rotate":
        layout = "TND" if case["packed"] else "BSND"
        how = dict(sections=_numbers(case["sections"]) or None, rotary_start=case["start"],
                   interleaved=case["interleaved"], layout=layout)
        out = []
        if case["ways"] != "grad":
            out.append(dsa.rotary_embedding(i["x"], i["positions"], i["freq"], **how))
        if case["ways"] != "forward":
            out.append(dsa.rotary_embedding_grad(i["d"], i["positions"], i["freq"], **how))
        return out
    if "plan" in state:
        got = state["plan"].run()
        return got if kind != "attend" or case["lse"] else got[0]
    if kind == "latent":
        return dsa.latent_cache_append(i["latent"], i["rope"], i["cache"], i["rope_cache"], i["table"], i["freq"],
                                       _kv_lengths(case), _query_lengths(case), norm_weight=i["weight"],
                                       interleaved=case["interleaved"], layout="TND")
    if kind == "index":
        return dsa.index_cache_append(i["keys"], i["cache"], i["table"], i["freq"], _kv_lengths(case),
                                      _query_lengths(case), norm_weight=i["weight"], norm_bias=i["bias"],
                                      interleaved=case["interleaved"], layout="TND")
    got = dsa.shared_prefix_attention(i["query"], i["cache"], i["cache"], i["table"], case["prefix"], _scale(case),
                                      _query_lengths(case), _kv_lengths(case), query_rope=i["query_rope"],
                                      key_rope=i["rope_cache"], layout_query="TND", return_softmax_lse=case["lse"])
    return got if case["lse"] else got[0]


# ------------------------------------------------------------------ the plain forms
def _cos_sin(positions, freq, sections):
    """cos and sin of each token's pairs, [..., rotary / 2], angles in 64 bits."""
    p = positions.double()
    if sections:
        pair_axis = torch.repeat_interleave(torch.arange(len(sections), device=p.device),
                                            torch.tensor(sections, device=p.device))
        p = p.movedim(0, -1)[..., pair_axis]
    else:
        p = p.unsqueeze(-1)
    angle = p * freq.double()
    return angle.cos().float(), angle.sin().float()


def _turned(x, cos, sin, interleaved):
    """The last dimension of x (32 bits) rotated pairwise; cos and sin are shared by the heads."""
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _rotate_plain(case, i):
    cos, sin = _cos_sin(i["positions"], i["freq"], _numbers(case["sections"]))
    lo, hi = case["start"], case["start"] + case["rotary"]

    def one(x, sin):
        y = x.float()
        return torch.cat([y[..., :lo], _turned(y[..., lo:hi], cos, sin, case["interleaved"]), y[..., hi:]], -1).to(x.dtype)

    out = []
    if case["ways"] != "grad":
        out.append(one(i["x"], sin))
    if case["ways"] != "forward":
        out.append(one(i["d"], -sin))
    return out


def _new_places(case, table):
    """(positions, cache rows) of the new tokens, in the order of the packed rows."""
    tokens, kv, page = _numbers(case["tokens"]), _numbers(case["kv"]), case["page"]
    dev = table.device
    t = torch.tensor(tokens, device=dev)
    b = torch.repeat_interleave(torch.arange(len(tokens), device=dev), t, output_size=sum(tokens))
    first = torch.tensor([k - n for k, n in zip(kv, tokens)], device=dev)
    within = torch.arange(sum(tokens), device=dev) - torch.tensor(_starts(tokens)[:-1], device=dev)[b]
    pos = first[b] + within
    return pos, table[b, pos // page].long() * page + pos % page


def _latent_plain(case, i):
    pos, rows = _new_places(case, i["table"])
    x = i["latent"].reshape(-1, case["dim"]).float()
    if case["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * i["weight"].float()
    cos, sin = _cos_sin(pos, i["freq"], None)
    r = _turned(i["rope"].reshape(-1, 1, ROPE).float(), cos, sin, case["interleaved"])
    i["cache"].view(-1, case["dim"])[rows] = x.to(i["cache"].dtype)
    i["rope_cache"].view(-1, ROPE)[rows] = r.reshape(-1, ROPE).to(i["cache"].dtype)
    return i["cache"], i["rope_cache"]


def _index_plain(case, i):
    pos, rows = _new_places(case, i["table"])
    n, w, r = case["heads"], case["width"], case["rotary"]
    x = i["keys"].reshape(-1, n, w).float()
    if case["norm"]:
        x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * i["weight"] + i["bias"]
    cos, sin = _cos_sin(pos, i["freq"], None)
    x = torch.cat([_turned(x[..., :r], cos, sin, case["interleaved"]), x[..., r:]], -1)
    i["cache"].view(-1, n, w)[rows] = x.to(i["cache"].dtype)
    return i["cache"]


def _cache_rows(table, page, first, last):
    t = torch.arange(first, last, device=table.device)
    return table[t // page].long() * page + t % page


def _attend_plain(case, i):
    d, n, prefix = case["dim"], case["heads"], case["prefix"]
    tokens, kv, page = _numbers(case["tokens"]), _numbers(case["kv"]), case["page"]
    q = torch.cat([i["query"], i["query_rope"]], -1).reshape(-1, n, d + ROPE)
    cache, rope = i["cache"].view(-1, d), i["rope_cache"].view(-1, ROPE)

    def keys(rows):
        return torch.cat([cache[rows], rope[rows]], -1).float()

    shared = keys(_cache_rows(i["table"][0], page, 0, prefix))
    out, tops, sums, at = [], [], [], 0
    for b, (t, total) in enumerate(zip(tokens, kv)):
        k = torch.cat([shared, keys(_cache_rows(i["table"][b], page, prefix, total))])
        s = (q[at:at + t].reshape(t * n, -1).float() @ k.t()).reshape(t, n, total) * _scale(case)
        if t > 1:
            seen = torch.arange(total, device=s.device) < torch.arange(total - t + 1, total + 1, device=s.device)[:, None]
            s = torch.where(seen[:, None], s, -math.inf)
        top = s.amax(-1)
        e = torch.exp(s - top[..., None])
        total_e = e.sum(-1)
        out.append((e.reshape(t * n, total) @ k[:, :d]).reshape(t, n, d) / total_e[..., None])
        tops.append(top)
        sums.append(total_e)
        at += t
    o = torch.cat(out).to(i["query"].dtype).reshape(i["query"].shape)
    if not case["lse"]:
        return o
    shape = (1, at, n) if case["packed"] else (len(tokens), 1, tokens[0], n)
    return o, torch.cat(tops).reshape(shape), torch.cat(sums).reshape(shape)


_PLAIN = dict(rotate=_rotate_plain, latent=_latent_plain, index=_index_plain, attend=_attend_plain)


# ------------------------------------------------------------------ sizes
def work(case):
    b = 4 if case["dtype"] == "fp32" else 2
    tokens = _numbers(case["tokens"])
    total, kind = sum(tokens), case["kind"]
    if kind == "rotate":
        passes = 2 if case["ways"] == "both" else 1
        axes = max(1, len(_numbers(case["sections"])))
        x = total * case["heads"]
        return {"bytes": passes * (2 * x * case["width"] * b + 8 * total * axes), "flops": passes * 3 * x * case["rotary"]}
    kv = _numbers(case["kv"])
    if kind in ("latent", "index"):
        width = case["dim"] + ROPE if kind == "latent" else case["heads"] * case["width"]
        pages = sum(-(-k // case["page"]) - (k - t) // case["page"] for t, k in zip(tokens, kv))
        return {"bytes": 2 * total * width * b + 4 * pages, "flops": total * width * 6}
    d, n, prefix = case["dim"], case["heads"], case["prefix"]
    seen = sum(t * k - t * (t - 1) // 2 for t, k in zip(tokens, kv))
    rows = prefix + sum(k - prefix for k in kv)
    stats = 8 * total * n if case["lse"] else 0
    return {"bytes": total * n * (2 * d + ROPE) * b + rows * (d + ROPE) * b + stats, "flops": 2 * seen * n * (2 * d + ROPE)}


# ------------------------------------------------------------------ 64 bits, from the definitions
def _rotation_matrices(positions, freq, axis_of_pair):
    """[tokens, pairs, 2, 2]: the rotation of each pair by position times frequency."""
    p = positions.double().reshape(-1, positions.shape[-1]) if axis_of_pair is None else positions.double()
    a = p.reshape(-1, 1) * freq.double() if axis_of_pair is None else p.reshape(p.shape[0], -1)[axis_of_pair].t() * freq.double()
    return torch.stack([torch.stack([a.cos(), -a.sin()], -1), torch.stack([a.sin(), a.cos()], -1)], -2)


def _exact_turn(x, m, interleaved):
    """x [tokens, heads, rotary] in 64 bits."""
    t, n, r = x.shape
    pairs = x.reshape(t, n, r // 2, 2) if interleaved else x.reshape(t, n, 2, r // 2).transpose(-1, -2)
    y = (m[:, None] * pairs.unsqueeze(-2)).sum(-1)
    return y.reshape(t, n, r) if interleaved else y.transpose(-1, -2).reshape(t, n, r)


def _exact_rotate(case, i):
    sections = _numbers(case["sections"])
    axis = torch.tensor([a for a, c in enumerate(sections) for _ in range(c)], device=i["x"].device) if sections else None
    m = _rotation_matrices(i["positions"], i["freq"], axis)
    lo, hi = case["start"], case["start"] + case["rotary"]

    def one(x, m):
        y = x.double().reshape(-1, case["heads"], case["width"])
        y[..., lo:hi] = _exact_turn(y[..., lo:hi].clone(), m, case["interleaved"])
        return y.reshape(x.shape)

    out = []
    if case["ways"] != "grad":
        out.append(one(i["x"], m))
    if case["ways"] != "forward":
        out.append(one(i["d"], m.transpose(-1, -2)))
    return out


def _exact_places(case, table):
    """(batch, position, block, slot) of each new token, one by one."""
    pages, got = table.tolist(), []
    for b, (t, k) in enumerate(zip(_numbers(case["tokens"]), _numbers(case["kv"]))):
        for p in range(k - t, k):
            got.append((p, pages[b][p // case["page"]], p % case["page"]))
    return [torch.tensor(v, device=table.device) for v in zip(*got)]


def _exact_latent(case, i):
    pos, block, slot = _exact_places(case, i["table"])
    x = i["latent"].double().reshape(-1, case["dim"])
    if case["norm"]:
        x = x / ((x * x).sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt() * i["weight"].double()
    r = _exact_turn(i["rope"].double().reshape(-1, 1, ROPE), _rotation_matrices(pos[None], i["freq"], None), case["interleaved"])
    cache, rope_cache = i["cache"].double(), i["rope_cache"].double()
    cache[block, slot, 0] = x
    rope_cache[block, slot, 0] = r[:, 0]
    return cache, rope_cache


def _exact_index(case, i):
    pos, block, slot = _exact_places(case, i["table"])
    w, r = case["width"], case["rotary"]
    x = i["keys"].double().reshape(-1, case["heads"], w)
    if case["norm"]:
        mean = x.sum(-1, keepdim=True) / w
        var = ((x - mean) ** 2).sum(-1, keepdim=True) / w
        x = (x - mean) / (var + 1e-6).sqrt() * i["weight"].double() + i["bias"].double()
    x[..., :r] = _exact_turn(x[..., :r].clone(), _rotation_matrices(pos[None], i["freq"], None), case["interleaved"])
    cache = i["cache"].double()
    cache[block, slot] = x
    return cache


def _exact_attend(case, i):
    d, n, page, prefix = case["dim"], case["heads"], case["page"], case["prefix"]
    tokens, kv = _numbers(case["tokens"]), _numbers(case["kv"])
    pages = i["table"].tolist()
    latents, ropes = i["cache"].reshape(-1, d), i["rope_cache"].reshape(-1, ROPE)
    q, qr = i["query"].reshape(-1, n, d), i["query_rope"].reshape(-1, n, ROPE)
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    top = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    total = torch.empty_like(top)
    row = 0
    for b, (t, length) in enumerate(zip(tokens, kv)):
        place = torch.tensor([pages[0 if p < prefix else b][p // page] * page + p % page for p in range(length)],
                             device=q.device)
        k, kr = latents[place].double(), ropes[place].double()
        step = max(1, 200_000_000 // (n * length))
        for r0 in range(0, t, step):
            r1 = min(t, r0 + step)
            s = (torch.matmul(q[row + r0:row + r1].double(), k.t()) + torch.matmul(qr[row + r0:row + r1].double(), kr.t())) * _scale(case)
            for r in range(r0, r1):   # row r of the sequence sees positions up to its own
                s[r - r0, :, length - t + r + 1:] = -math.inf
            a = slice(row + r0, row + r1)
            top[a] = s.max(-1).values
            e = torch.exp(s - top[a].unsqueeze(-1))
            total[a] = e.sum(-1)
            out[a] = torch.matmul(e, k) / total[a].unsqueeze(-1)
        row += t
    out = out.reshape(i["query"].shape)
    if not case["lse"]:
        return out
    shape = (1, row, n) if case["packed"] else (len(tokens), 1, tokens[0], n)
    return out, top.reshape(shape), total.reshape(shape)


def exact(case, seed):
    i = _inputs(case, seed)
    return dict(rotate=_exact_rotate, latent=_exact_latent, index=_exact_index, attend=_exact_attend)[case["kind"]](case, i)
