"""Values that are not finite in keys and values: which outputs and gradients they have to reach, case by case."""
import math

import pytest
import torch

from tests.test_dense_attention_gpu import BF, HF, call, make
from tests.test_dense_attention_grad_gpu import gradients

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("what", ["key", "value", "key_rope"])
@pytest.mark.parametrize("mode", [0, 3])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_reach(what, value, mode, splits, dtype):
    """Token 150 of key head 1, whole: seen by the queries from 150 on (mode 3), or by all, of heads 2 and 3.

    Key: every product with it is NaN (of 128 or 64 infinities with queries of both signs too), and so are those
    queries' statistics and all of their P: every token's d_key, d_key_rope and d_value of that head.
    Value: P does not know it, so d_value is as without it; dP and delta of those queries are NaN (d_out has both signs),
    and so are all of their dS: every token's d_key and d_key_rope."""
    tokens = [50, 200]
    t = make(dtype, 4, 2, 128, 64, tokens, tokens, False, 40, behind=3)
    t = {k: v.clone() for k, v in t.items()}
    do = make(dtype, 4, 4, 128, 0, tokens, tokens, False, 41, behind=3)["query"]
    clean = gradients(t, do, call(t, tokens, tokens, False, 0.1, mode), tokens, tokens, False, 0.1, mode, splits=splits)
    t[what][1, 150, 1] = value
    got = gradients(t, do, call(t, tokens, tokens, False, 0.1, mode), tokens, tokens, False, 0.1, mode, splits=splits)
    first = 150 if mode == 3 else 0
    dq, dk, dv, dqr, dkr = got
    for x in (dq, dqr):
        assert not torch.isfinite(x[1, first:200, 2:]).any()
    for x in (dk, dkr) + ((dv,) if what != "value" else ()):
        assert not torch.isfinite(x[1, :200, 1]).any()
    if what == "value":
        assert torch.equal(dv, clean[2])
    for x, y in zip(got, clean):   # the other sequence and head, and the padding
        assert torch.equal(x[0], y[0]) and not x[1, 200:].any()
    for x, y in ((dq, clean[0]), (dqr, clean[3])):
        assert torch.equal(x[1, :first], y[1, :first]) and torch.equal(x[1, :, :2], y[1, :, :2])
    for x, y in zip(got[1:3] + got[4:], clean[1:3] + clean[4:]):
        assert torch.equal(x[1, :, 0], y[1, :, 0])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [math.nan, -math.inf])
@pytest.mark.parametrize("mode", [0, 3])
@pytest.mark.parametrize("n1,n2,d,dr,tokens,splits", [(4, 2, 128, 64, [50, 200], 1), (4, 2, 64, 0, [50, 200], 3), (4, 2, 128, 0, [70, 200], 0),
                                                      (32, 8, 128, 0, [900, 1400], 1), (32, 8, 128, 64, [900, 1400], 1),
                                                      (32, 8, 64, 0, [900, 1400], 1)])
def test_statistics_do_not_know_the_values(n1, n2, d, dr, tokens, splits, mode, value, dtype):
    """sm_max and sm_sum are of the scores; the output of each row that sees the value is not finite, in that column at least"""
    t = make(dtype, n1, n2, d, dr, tokens, tokens, False, 42, behind=3)
    want = call(t, tokens, tokens, False, 0.1, mode, kv_splits=splits)
    t["value"] = t["value"].clone()
    t["value"][1, 150, 1, 7] = value
    got = call(t, tokens, tokens, False, 0.1, mode, kv_splits=splits)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    first, per = 150 if mode == 3 else 0, n1 // n2
    assert not torch.isfinite(got[0][1, first:tokens[1], per:2 * per, 7]).any()
    assert torch.equal(got[0][1, :first], want[0][1, :first]) and torch.equal(got[0][0], want[0][0])
    assert torch.equal(got[0][1, :, :per], want[0][1, :, :per]) and torch.equal(got[0][1, :, 2 * per:], want[0][1, :, 2 * per:])
