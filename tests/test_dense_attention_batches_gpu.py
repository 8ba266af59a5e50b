"""dense_attention and its gradient on padded batches whose sequences lie apart: the same results as on copies of
them, and plans that read what was written since."""
import pytest
import torch

import dsa_triton_ascend_amd as dsa
from tests.test_dense_attention_gpu import BF, HF, call, make
from tests.test_dense_attention_grad_gpu import gradients

pytestmark = pytest.mark.gpu


def lie(x, how):
    """x's values in a tensor of its shape that lies as `how` says"""
    B, S, N, D = x.shape
    if how == "longer":          # the filled part of a cache
        y = torch.full((B, S + 37, N, D), float("nan"), dtype=x.dtype, device=x.device)[:, 11:11 + S]
    elif how == "heads first":   # [B, N, S, D] underneath
        y = torch.empty(B, N, S, D, dtype=x.dtype, device=x.device).transpose(1, 2)
    elif how == "both":          # heads first, in a longer cache
        y = torch.full((B, N, S + 5, D), float("nan"), dtype=x.dtype, device=x.device)[:, :, :S].transpose(1, 2)
    else:                        # batches backwards: none of the strides order the others
        y = torch.empty(S, B, N, D, dtype=x.dtype, device=x.device).transpose(0, 1)
    return y.copy_(x)


HOW = ["longer", "heads first", "both", "rows first"]
CASES = [  # n1, n2, d, dr, tokens, kv, mode
    (4, 2, 128, 64, [80, 41, 1], [95, 60, 33], 3),
    (6, 2, 64, 0, [33, 0, 70], [33, 20, 70], 0),       # (a group of three)
    (32, 4, 128, 0, [1, 1, 1], [500, 1, 1333], 3),     # single tokens
    (5, 1, 128, 0, [300, 257], [300, 511], 3),
    (16, 16, 64, 0, [1200, 1100], [1300, 1100], 3),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_same_as_on_copies(case, how, dtype):
    n1, n2, d, dr, tokens, kv, mode = CASES[case]
    t = make(dtype, n1, n2, d, dr, tokens, kv, False, 80 + case)
    do = make(dtype, n1, n1, d, 0, tokens, tokens, False, 90 + case)["query"]
    apart = {k: None if v is None else lie(v, how) for k, v in t.items()}
    want, got = (call(x, tokens, kv, False, 0.1, mode) for x in (t, apart))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = gradients(t, do, want, tokens, kv, False, 0.1, mode)
    for x, g, o in ((apart, lie(do, how), lie(want[0], how)), (t, lie(do, how), want[0]), ({**t, "key": apart["key"]}, do, want[0])):
        again = gradients(x, g, (o,) + tuple(want[1:]), tokens, kv, False, 0.1, mode)
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(again, grads))


def test_shared_by_the_batch():
    """One prompt's keys for several sequences, expanded over the batch"""
    t = make(BF, 4, 2, 128, 64, [40, 40, 7], [90, 90, 90], False, 95)
    for k in ("key", "value", "key_rope"):
        t[k] = t[k][:1].expand(3, *t[k].shape[1:])
    got = call(t, [40, 40, 7], [90, 90, 90], False, 0.1)
    want = call({k: v.contiguous() for k, v in t.items()}, [40, 40, 7], [90, 90, 90], False, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("captured", [False, True])
def test_plans_read_what_was_written_since(how, captured):
    tokens, kv = [1, 1, 1], [900, 1400, 333]
    t = make(BF, 16, 2, 128, 0, tokens, kv, False, 50)
    apart = {k: None if v is None else lie(v, how) for k, v in t.items()}
    do = make(BF, 16, 16, 128, 0, tokens, tokens, False, 51)["query"]
    plan = dsa.DenseAttentionPlan(apart["query"], apart["key"], apart["value"], 0.1, tokens, kv, return_softmax_lse=True)
    d_out = lie(do, how)
    out, mx, sm = plan.run()
    back = dsa.DenseAttentionGradPlan(apart["query"], apart["key"], apart["value"], d_out, out, mx, sm, 0.1,
                                      actual_seq_lengths_query=tokens, actual_seq_lengths_kv=kv)

    def both():
        return plan.run() + back.run()[:3]

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both()
    for seed in (52, 53, 54):
        t2 = make(BF, 16, 2, 128, 0, tokens, kv, False, seed)
        do2 = make(BF, 16, 16, 128, 0, tokens, tokens, False, seed + 100)["query"]
        for k in ("query", "key", "value"):
            apart[k].copy_(t2[k])
        d_out.copy_(do2)
        if captured:
            graph.replay()
        else:
            got = both()
        torch.cuda.synchronize()
        fwd = call(t2, tokens, kv, False, 0.1)
        want = tuple(fwd) + tuple(gradients(t2, do2, fwd, tokens, kv, False, 0.1)[:3])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_sequences_far_apart():
    """Sequences 2^31 elements from each other, rows of 2^23: offsets past 32 bits in both"""
    wide = torch.empty(2, 300, 1 << 23, dtype=BF, device="cuda")
    t = make(BF, 2, 1, 128, 0, [256, 250], [256, 250], False, 60)
    want = call(t, [256, 250], [256, 250], False, 0.1)
    for what, at in (("key", 0), ("value", 1024)):
        far = wide[:, 20:276, at:at + 128].unsqueeze(2)
        far.copy_(t[what])
        t[what] = far
    got = call(t, [256, 250], [256, 250], False, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_a_plan_copies_is_written_in_the_plan():
    """Strides within the last dimension: the documented copy, and the others in place beside it"""
    t = make(BF, 4, 2, 128, 0, [50, 20], [70, 64], False, 55)
    wide = torch.empty(2, 70, 2, 256, dtype=BF, device="cuda")
    key = wide[..., ::2].copy_(t["key"])
    plan = dsa.DenseAttentionPlan(t["query"], key, lie(t["value"], "longer"), 0.1, [50, 20], [70, 64], return_softmax_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(plan.run(), call(t, [50, 20], [70, 64], False, 0.1)))
    t["key"] = make(BF, 4, 2, 128, 0, [50, 20], [70, 64], False, 56)["key"]
    plan.k.copy_(t["key"].flatten(0, 1))
    assert all(torch.equal(a, b) for a, b in zip(plan.run(), call(t, [50, 20], [70, 64], False, 0.1)))
