"""Dense attention of whole prompts and layer norm, forward and backward, as measured cases.

``listed()`` holds the fixed cases, ``draw(rng)`` gives further ones of the same ranges. ``prepare``
makes what a program has in hand before the call, ``run`` is one pass: with ``own`` the package's
operators, else the same operators written out in elementary torch. ``exact`` computes a case's
outputs in 64 bits from the definitions, apart from both.

Kinds of case:
  attend      ``dense_attention``: every head of a prompt (or of a chunk of one, or of a single new token)
              over keys and values of its group, causal
  train       the same and ``dense_attention_grad``: output and all gradients of a training step
  norm        ``layer_norm`` of an indexer's keys or of a model's hidden rows
  norm_train  the same and ``layer_norm_grad``
"""
import math

import torch

own = False

ROPE = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _numbers(text):
    return [int(v) for v in text.split(",") if v]


def _text(values):
    return ",".join(str(int(v)) for v in values)


def listed():
    return [
        # the smallest call: one short prompt, few narrow heads; launch and host time count
        dict(name="attend_small", kind="attend", dtype="bf16", tokens="60", kv="60", packed=True, heads=8, groups=2,
             dim=64, rope=0, causal=True, lse=False),
        # one new token for each of four sequences over long ragged keys, 32 heads on 4 key heads
        dict(name="attend_token", kind="attend", dtype="bf16", tokens="1,1,1,1", kv="4000,8190,6001,7311", packed=False,
             heads=32, groups=4, dim=128, rope=0, causal=True, lse=False),
        # a padded batch of prompts, narrow heads, a key head each; no causal mask (an encoder's pass)
        dict(name="attend_padded", kind="attend", dtype="fp16", tokens="777,512,640,130", kv="777,512,640,130",
             packed=False, heads=16, groups=16, dim=64, rope=0, causal=False, lse=False),
        # a chunk of a long prompt, after what is in the keys already, 32 heads on 8
        dict(name="attend_chunk", kind="attend", dtype="bf16", tokens="2048", kv="14001", packed=True, heads=32,
             groups=8, dim=128, rope=0, causal=True, lse=False),
        # packed ragged prompts with the latent expanded to keys and values of each head, rotary part shared by
        # the heads; the statistics that the indexer's dense loss takes
        dict(name="attend_prompts", kind="attend", dtype="bf16", tokens="1024,2000,5168", kv="1024,2000,5168",
             packed=True, heads=32, groups=32, dim=128, rope=64, causal=True, lse=True),
        # training on packed short samples, narrow heads in fp16
        dict(name="train_short", kind="train", dtype="fp16", tokens="200,77,333,1,150", kv="200,77,333,1,150",
             packed=True, heads=8, groups=4, dim=64, rope=0, causal=True, lse=False),
        # a training step's attention over one long sample, 32 heads on 8
        dict(name="train_long", kind="train", dtype="bf16", tokens="8192", kv="8192", packed=True, heads=32, groups=8,
             dim=128, rope=0, causal=True, lse=False),
        # and of two ragged samples with rotary parts beside every head
        dict(name="train_rope", kind="train", dtype="bf16", tokens="4093,2100", kv="4093,2100", packed=True, heads=16,
             groups=16, dim=128, rope=64, causal=True, lse=False),
        # an indexer's keys in a decode step
        dict(name="norm_decode", kind="norm", dtype="bf16", rows=48, width=128, extra=0, weights="fp32"),
        # an indexer's keys of packed prompts, a slice of a wider projection
        dict(name="norm_keys", kind="norm", dtype="bf16", rows=18216, width=128, extra=64, weights="fp32"),
        # the hidden rows of a training batch, with all gradients
        dict(name="norm_hidden", kind="norm_train", dtype="bf16", rows=16383, width=4096, extra=0, weights="bf16"),
        # odd widths in 32 bits
        dict(name="norm_odd", kind="norm_train", dtype="fp32", rows=5003, width=1001, extra=0, weights="fp32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _parts(rng, total, most):
    """`total` tokens as up to `most` sequences of uneven lengths."""
    n = min(rng.randint(1, most), total)
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    kind = rng.choice(["attend", "attend", "train", "train", "norm", "norm_train"])
    if kind in ("norm", "norm_train"):
        width = rng.choice([64, 128, 128, 256, 1024, 4096, 5120, rng.randint(1, 1500), rng.randint(1500, 9000)])
        rows = _log(rng, 1, min(40000, 60_000_000 // width))
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rows=rows, width=width,
                    extra=rng.choice([0, 0, 64, 7]), weights=rng.choice(["same", "fp32"]))
    dim, rope = rng.choice([(64, 0), (128, 0), (128, 0), (128, 64)])
    groups, per = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4, 8])
    heads = groups * per
    causal = rng.random() < 0.8
    work = 4e8 if kind == "train" else 1.6e9   # pairs of a query row and a key, over all heads
    if kind == "attend" and rng.random() < 0.35:   # single tokens, or a few, over long keys
        n, s = _log(rng, 1, 48), rng.choice([1, 1, 1, 2, 4])
        tokens = [s] * n
        most = max(64, min(16000, int(work / 8 / (n * s * heads))))
        kv = [max(s, _log(rng, 16, most)) for _ in range(n)]
        packed = False
    else:
        packed = rng.random() < 0.7
        longest = int(min(8192, math.sqrt(work / heads)))
        total = _log(rng, 8, longest)
        tokens = _parts(rng, total, 6 if packed else 4)
        if rng.random() < 0.3:   # chunks after what the keys hold already
            kv = [t + rng.randint(0, max(1, longest - total)) for t in tokens]
        else:
            kv = list(tokens)
    return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16"]), tokens=_text(tokens), kv=_text(kv), packed=packed,
                heads=heads, groups=groups, dim=dim, rope=rope, causal=causal, lse=kind == "attend" and rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
class _Source:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(seed)

    def normal(self, shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=self.g, device=self.dev, dtype=torch.float32) * scale).to(dtype)


def _starts(lengths):
    out = [0]
    for v in lengths:
        out.append(out[-1] + v)
    return out


def _lead(lengths, packed):
    return (sum(lengths),) if packed else (len(lengths), max(lengths))


def _inputs(case, seed):
    s, dt = _Source(seed), DTYPES[case["dtype"]]
    if case["kind"] in ("norm", "norm_train"):
        rows, width = case["rows"], case["width"]
        wdt = dt if case["weights"] in ("same", case["dtype"]) else torch.float32
        x = (s.normal((rows, width + case["extra"]), dt, 1.5) + 0.25)[:, :width]
        return dict(x=x, d=s.normal((rows, width), dt), weight=(1 + 0.1 * s.normal((width,), torch.float32)).to(wdt),
                    bias=s.normal((width,), torch.float32, 0.1).to(wdt))
    tokens, kv, packed = _numbers(case["tokens"]), _numbers(case["kv"]), case["packed"]
    n, g, d = case["heads"], case["groups"], case["dim"]
    q_lead, k_lead = _lead(tokens, packed), _lead(kv, packed)
    i = dict(query_rope=None, key_rope=None)
    if case["rope"]:   # keys and values side by side out of one projection, one rotary key for all heads
        both = s.normal(k_lead + (g, 2 * d), dt)
        i.update(query=s.normal(q_lead + (n, d), dt), key=both[..., :d], value=both[..., d:],
                 query_rope=s.normal(q_lead + (n, ROPE), dt),
                 key_rope=s.normal(k_lead + (1, ROPE), dt).expand(*k_lead, g, ROPE))
    elif tokens == kv:   # one projection for queries, keys and values
        all_ = s.normal(q_lead + (n + 2 * g, d), dt)
        i.update(query=all_[..., :n, :], key=all_[..., n:n + g, :], value=all_[..., n + g:, :])
    else:
        i.update(query=s.normal(q_lead + (n, d), dt), key=s.normal(k_lead + (g, d), dt), value=s.normal(k_lead + (g, d), dt))
    if case["kind"] == "train":
        i["d_out"] = s.normal(q_lead + (n, d), dt)
    return i


def _scale(case):
    return 1.0 / math.sqrt(case["dim"] + case["rope"])


def _how(case, i):
    """The keyword arguments of both attention calls."""
    tokens, kv = _numbers(case["tokens"]), _numbers(case["kv"])
    if case["packed"]:
        tokens, kv = _starts(tokens)[1:], _starts(kv)[1:]
    return dict(scale_value=_scale(case), actual_seq_lengths_query=tokens, actual_seq_lengths_kv=kv,
                query_rope=i["query_rope"], key_rope=i["key_rope"], layout="TND" if case["packed"] else "BSND",
                sparse_mode=3 if case["causal"] else 0)


def prepare(case, seed):
    i = _inputs(case, seed)
    state = dict(case=case, i=i)
    if own and case["kind"] == "attend" and not case["packed"]:   # a serving loop keeps the plan of its step
        import dsa_triton_ascend_amd as dsa
        state["plan"] = dsa.DenseAttentionPlan(i["query"], i["key"], i["value"], return_softmax_lse=case["lse"],
                                               **_how(case, i))
    return state


def run(state):
    case, i = state["case"], state["i"]
    if not own:
        return _PLAIN[case["kind"]](case, i)
    import dsa_triton_ascend_amd as dsa
    kind = case["kind"]
    if kind == "norm":
        return dsa.layer_norm(i["x"], i["weight"], i["bias"])
    if kind == "norm_train":
        y, mean, rstd = dsa.layer_norm(i["x"], i["weight"], i["bias"], return_stats=True)
        return (y,) + dsa.layer_norm_grad(i["d"], i["x"], mean, rstd, i["weight"], i["bias"])
    if kind == "attend":
        if "plan" in state:
            got = state["plan"].run()
        else:
            got = dsa.dense_attention(i["query"], i["key"], i["value"], return_softmax_lse=case["lse"], **_how(case, i))
        return got if case["lse"] else got[0]
    how = _how(case, i)
    out, top, total = dsa.dense_attention(i["query"], i["key"], i["value"], return_softmax_lse=True, **how)
    grads = dsa.dense_attention_grad(i["query"], i["key"], i["value"], i["d_out"], out, top, total, **how)
    return (out,) + tuple(g for g in grads if g is not None)


# ------------------------------------------------------------------ the plain forms
NORM_EPS = 1e-6


def _norm_plain(case, i, train=False):
    x = i["x"].float()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt(c.square().mean(-1, keepdim=True) + NORM_EPS)
    hat = c * rstd
    w = i["weight"].float()
    y = (hat * w + i["bias"].float()).to(i["x"].dtype)
    if not train:
        return y
    d = i["d"].float()
    g = d * w
    dx = (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True)) * rstd
    wdt = i["weight"].dtype
    return y, dx.to(y.dtype), (d * hat).sum(0).to(wdt), d.sum(0).to(wdt)


def _norm_train_plain(case, i):
    return _norm_plain(case, i, True)


def _sequence(case, x, b, lengths):
    """Sequence b's rows [length, heads, width] of a packed or padded tensor."""
    if not case["packed"]:
        return x[b, :lengths[b]]
    at = _starts(lengths)[b]
    return x[at:at + lengths[b]]


def _joined(case, i, which):
    x, r = i[which], i[which + "_rope"]
    return x if r is None else torch.cat([x, r], -1)


def _seen(case, t, k, r0, r1, dev):
    """[rows, keys]: which keys the query rows r0 .. r1 of a sequence see."""
    return torch.arange(k, device=dev) < torch.arange(k - t + r0 + 1, k - t + r1 + 1, device=dev)[:, None]


def _chunks(t, per_row):
    step = max(1, (1 << 28) // max(1, per_row))
    return [(r, min(t, r + step)) for r in range(0, t, step)]


def _attention_plain(case, i, train=False):
    tokens, kv = _numbers(case["tokens"]), _numbers(case["kv"])
    n, g, d, scale = case["heads"], case["groups"], case["dim"], _scale(case)
    per, wide = n // g, d + case["rope"]
    q_all, k_all = _joined(case, i, "query"), _joined(case, i, "key")
    dev = q_all.device
    z = lambda like, width: torch.zeros(like.shape[:-1] + (width,), dtype=torch.float32, device=dev)
    out = z(q_all, d)
    top, total = (torch.zeros(q_all.shape[:-1], dtype=torch.float32, device=dev) for _ in range(2))
    if train:
        dq_all, dk_all, dv_all = z(q_all, wide), z(k_all, wide), z(k_all, d)
    for b, (t, length) in enumerate(zip(tokens, kv)):
        q_b, o_b, top_b, sum_b = (_sequence(case, x, b, tokens) for x in (q_all, out, top, total))
        k_b, v_b = (_sequence(case, x, b, kv) for x in (k_all, i["value"]))
        if train:
            dq_b, do_b = (_sequence(case, x, b, tokens) for x in (dq_all, i["d_out"]))
            dk_b, dv_b = (_sequence(case, x, b, kv) for x in (dk_all, dv_all))
        for h in range(g):
            own_heads = slice(h * per, (h + 1) * per)
            k, v = k_b[:, h].float(), v_b[:, h].float()
            for r0, r1 in _chunks(t, per * length):
                q = q_b[r0:r1, own_heads].float().reshape(-1, wide)
                s = (q @ k.t()).reshape(r1 - r0, per, length) * scale
                if case["causal"]:
                    seen = _seen(case, t, length, r0, r1, dev)[:, None]
                    s = torch.where(seen, s, -math.inf)
                m = s.amax(-1, keepdim=True)
                e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
                l = e.sum(-1, keepdim=True)
                p = (e / torch.where(l == 0, 1.0, l)).reshape(-1, length)
                o = p @ v
                o_b[r0:r1, own_heads] = o.reshape(r1 - r0, per, d)
                top_b[r0:r1, own_heads] = torch.where(l == 0, 0.0, m)[..., 0]
                sum_b[r0:r1, own_heads] = l[..., 0]
                if not train:
                    continue
                do = do_b[r0:r1, own_heads].float().reshape(-1, d)
                ds = p * (do @ v.t() - (do * o).sum(-1, keepdim=True)) * scale
                dq_b[r0:r1, own_heads] = (ds @ k).reshape(r1 - r0, per, wide)
                dk_b[:, h] += ds.t() @ q
                dv_b[:, h] += p.t() @ do
    dt = i["query"].dtype
    out = out.to(dt)
    if train:
        return (out,) + _parted(case, dq_all.to(dt), dk_all.to(dt), dv_all.to(dt))
    return (out, _stat(case, top), _stat(case, total)) if case["lse"] else out


def _parted(case, dq, dk, dv):
    d = case["dim"]
    if not case["rope"]:
        return dq, dk, dv
    return dq[..., :d], dk[..., :d], dv, dq[..., d:], dk[..., d:]


def _stat(case, x):
    """[.., tokens, heads] as the statistics are laid out: [B, groups, S, heads a group], or [groups, T, ..]."""
    return x.unflatten(-1, (case["groups"], -1)).movedim(-2, -3).contiguous()


def _train_plain(case, i):
    return _attention_plain(case, i, True)


_PLAIN = dict(attend=_attention_plain, train=_train_plain, norm=_norm_plain, norm_train=_norm_train_plain)


# ------------------------------------------------------------------ sizes
def work(case):
    b = 4 if case["dtype"] == "fp32" else 2
    kind = case["kind"]
    if kind in ("norm", "norm_train"):
        x = case["rows"] * case["width"]
        if kind == "norm":
            return {"bytes": 2 * x * b, "flops": 7 * x}
        return {"bytes": 5 * x * b, "flops": 22 * x}   # x twice: it does not fit the caches between the passes
    tokens, kv = _numbers(case["tokens"]), _numbers(case["kv"])
    n, g, d, wide = case["heads"], case["groups"], case["dim"], case["dim"] + case["rope"]
    pairs = 0
    for t, k in zip(tokens, kv):
        if not case["causal"]:
            pairs += t * k
        else:
            first = max(0, t - k)   # rows before that see nothing
            rows = t - first
            pairs += rows * k - rows * (rows - 1) // 2
    rows, keys = sum(tokens), sum(kv)
    forward = {"bytes": b * (rows * n * (wide + d) + keys * (g * 2 * d + case["rope"])) + (8 * rows * n if case["lse"] else 0),
               "flops": 2 * pairs * n * (wide + d)}
    if kind == "attend":
        return forward
    # the gradients' own four products, and the scores once more: P would be more bytes than its product takes
    return {"bytes": b * (rows * n * (3 * wide + 3 * d) + keys * g * (3 * wide + 3 * d)),
            "flops": forward["flops"] + 2 * pairs * n * (3 * wide + 2 * d)}


# ------------------------------------------------------------------ 64 bits, from the definitions
def _exact_norm(case, i):
    x, w, bias = i["x"].double(), i["weight"].double(), i["bias"].double()
    n = case["width"]
    mean = x.sum(-1) / n
    var = ((x - mean[:, None]) ** 2).sum(-1) / n
    std = (var + NORM_EPS).sqrt()
    y = (x - mean[:, None]) / std[:, None] * w + bias
    if case["kind"] == "norm":
        return y
    # d y_j / d x_k = w_j / std (delta_jk - 1/n - (x_j - mean)(x_k - mean) / (n std^2))
    d = i["d"].double()
    a = (d * w).sum(-1) / n
    c = (d * w * (x - mean[:, None])).sum(-1) / n / std ** 2
    dx = (d * w - a[:, None] - (x - mean[:, None]) * c[:, None]) / std[:, None]
    return y, dx, (d * (x - mean[:, None]) / std[:, None]).sum(0), d.sum(0)


def _exact_attention(case, i):
    tokens, kv = _numbers(case["tokens"]), _numbers(case["kv"])
    n, g, d, wide, train = case["heads"], case["groups"], case["dim"], case["dim"] + case["rope"], case["kind"] == "train"
    dev = i["query"].device
    new = lambda lead, heads, width: torch.zeros(lead + (heads, width), dtype=torch.float64, device=dev)
    q_lead, k_lead = _lead(tokens, case["packed"]), _lead(kv, case["packed"])
    out, dq, dk, dv = new(q_lead, n, d), new(q_lead, n, wide), new(k_lead, g, wide), new(k_lead, g, d)
    top, total = new(q_lead, n, 1), new(q_lead, n, 1)
    for h in range(n):
        for b, (t, length) in enumerate(zip(tokens, kv)):
            if case["packed"]:
                qs, ks = slice(sum(tokens[:b]), sum(tokens[:b + 1])), slice(sum(kv[:b]), sum(kv[:b + 1]))
            else:
                qs, ks = (b, slice(0, t)), (b, slice(0, length))
            at = lambda rows, head: (rows + (head,)) if isinstance(rows, tuple) else (rows, head)
            group = h // (n // g)
            q, k, v = i["query"][at(qs, h)].double(), i["key"][at(ks, group)].double(), i["value"][at(ks, group)].double()
            if case["rope"]:
                q = torch.cat([q, i["query_rope"][at(qs, h)].double()], 1)
                k = torch.cat([k, i["key_rope"][at(ks, group)].double()], 1)
            s = torch.mm(q, k.t()).mul_(_scale(case))
            if case["causal"]:   # query row r is token length - t + r
                s.masked_fill_(torch.ones(t, length, dtype=torch.bool, device=dev).triu_(length - t + 1), -math.inf)
            empty = s[:, 0] == -math.inf   # (causal: what sees any key sees the first)
            m = s.max(1).values.masked_fill_(empty, 0.0)
            p = s.sub_(m[:, None]).exp_()
            l = p.sum(1)
            top[at(qs, h)], total[at(qs, h)] = m[:, None], l[:, None]
            p /= l.masked_fill(empty, 1.0)[:, None]
            out[at(qs, h)] = torch.mm(p, v)
            if not train:
                continue
            do = i["d_out"][at(qs, h)].double()
            dv[at(ks, group)] += torch.mm(p.t(), do)
            dp = torch.mm(do, v.t())
            dp -= (p * dp).sum(1, keepdim=True)
            ds = dp.mul_(p).mul_(_scale(case))
            dq[at(qs, h)] = torch.mm(ds, k)
            dk[at(ks, group)] += torch.mm(ds.t(), q)
    if train:
        return (out,) + _parted(case, dq, dk, dv)
    if not case["lse"]:
        return out
    lay = lambda x: x.reshape(q_lead + (g, n // g)).transpose(-2, -3).contiguous()
    return out, lay(top), lay(total)


def exact(case, seed):
    i = _inputs(case, seed)
    return _exact_norm(case, i) if case["kind"] in ("norm", "norm_train") else _exact_attention(case, i)
