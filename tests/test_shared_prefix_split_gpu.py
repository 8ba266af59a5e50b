"""shared_prefix_attention where the shared tokens are cut into items of their own, for the head rows of all
sequences, beside the sequences' own items: each width of such items (32, 64, 128 head rows) and each D.

The form that a call takes is the library's choice, so every test asserts it, from the workspace bytes: p prefix
ranges and o own ones take 16 m (p + o) bytes of statistics (m head rows, to 256 bytes) and p blocks_p + o blocks_o
blocks of 32 rows of D floats. Tolerances are test_shared_prefix_gpu's."""
import pytest
import torch

import dsa_triton_ascend_amd as dsa

from .test_shared_prefix_gpu import BF, check, exact, make

pytestmark = pytest.mark.gpu
# width of the prefix items: heads, sequences (head rows that fill no whole item)
WIDTHS = {32: (4, 6), 64: (8, 7), 128: (16, 41)}


def ranges(plan):
    """(prefix ranges, own ranges) of a plan's run()"""
    batch, m, d, nbytes = plan.batch, plan.total_rows * plan.n1, plan.d, plan.ws_bytes
    mt = 4 if m > 64 else 2 if m > 32 else 1
    blocks_p, blocks_o = -(-m // (32 * mt)) * mt, m // 32 + batch + 1
    if nbytes == 0:
        return 0, 1
    got = [(p, o) for p in range(193 if plan.prefix else 1) for o in range(1, 257)
           if -(-16 * m * (p + o) // 256) * 256 + (p * blocks_p + o * blocks_o) * 128 * d == nbytes]
    assert len(got) == 1, got
    return got[0]


def plan_of(t, tokens, kv, prefix, scale, mode=3, splits=0, least=1):
    plan = dsa.SharedPrefixPlan(t["q"], t["k"], t["k"], t["table"], prefix, scale, tokens, kv, t["qr"], t["kr"],
                                sparse_mode=mode, return_softmax_lse=True, kv_splits=splits)
    p, o = ranges(plan)
    assert p >= least, f"{p} prefix ranges, {o} own ones: not the form that this test is about"
    return plan


def lengths(batch, prefix):
    """One token a sequence; sequences that end inside the prefix, at its end, at a range's end, and an empty one"""
    kv = [prefix + 1 + 13 * b for b in range(batch)]
    kv[0], kv[2], kv[3], kv[-1] = 0, prefix, 128, prefix - 37
    return kv


@pytest.mark.parametrize("width", WIDTHS)
def test_ranges_of_nan_only(width):
    """A range of tokens none of whose scores is a number makes the rows that see it NaN, as the formula does,
    though it has no maximum to weigh it by; rows that do not see it keep their values."""
    n1, batch = WIDTHS[width]
    prefix, page = 1024, 32
    kv = lengths(batch, prefix)
    t = make(BF, n1, 128, [1] * batch, kv, prefix, page, False, 560)
    want = exact(t, [1] * batch, kv, prefix, 0.04, 3, False)
    poisoned = t["table"][0, 12:24].long()   # tokens 384 to 767: whole ranges of 96 as of 128
    t["k"][poisoned], t["kr"][poisoned] = float("nan"), float("nan")
    got = plan_of(t, None, kv, prefix, 0.04, least=4).run()
    for b in range(batch):
        if kv[b] <= 384:
            check(got, want, rows=slice(b, b + 1))
        else:
            assert torch.isnan(got[0][b]).all() and torch.isnan(got[2][b]).all()


@pytest.mark.parametrize("prefix,first,last", [(0, 256, 768), (260, 388, 772)])
def test_own_ranges_of_nan_only(prefix, first, last):
    """The same in the middle of one sequence's own tokens, cut into ranges of 256 or 128."""
    kv = [1100, 1000, 90]
    t = make(BF, 16, 128, [1] * 3, kv, prefix, 4, False, 570)
    want = exact(t, [1] * 3, kv, prefix, 0.04, 3, False)
    poisoned = t["table"][1, first // 4:last // 4].long()
    t["k"][poisoned] = float("nan")
    got = plan_of(t, None, kv, prefix, 0.04, splits=8, least=0).run()
    assert torch.isnan(got[0][1]).all()
    for b in (0, 2):
        check(got, want, rows=slice(b, b + 1))
