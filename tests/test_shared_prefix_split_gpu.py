"""shared_prefix_attention where the shared tokens are cut into items of their own, for the head rows of all
sequences, beside the sequences' own items: each width of such items (32, 64, 128 head rows) and each D.

The form that a call takes is the library's choice, so every test asserts it, from the workspace bytes: p prefix
ranges and o own ones take 16 m (p + o) bytes of statistics (m head rows, to 256 bytes) and p blocks_p + o blocks_o
blocks of 32 rows of D floats. Tolerances are test_shared_prefix_gpu's."""
import math

import pytest
import torch

import dsa_triton_ascend_amd as dsa

from .test_shared_prefix_gpu import BF, HF, check, exact, make

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


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [128, 256, 512])
@pytest.mark.parametrize("width", WIDTHS)
def test_against_formula(width, d, dtype):
    """The prefix through table row 0, of a sequence that has no token itself."""
    n1, batch = WIDTHS[width]
    prefix = 1031
    kv = lengths(batch, prefix)
    t = make(dtype, n1, d, [1] * batch, kv, prefix, 16, False, 500 + d)
    scale = 1 / math.sqrt(d + 64)
    check(plan_of(t, None, kv, prefix, scale).run(), exact(t, [1] * batch, kv, prefix, scale, 3, False))


@pytest.mark.parametrize("n1,batch,d", [(2, 5, 128), (2, 5, 512), (4, 5, 128), (4, 5, 512), (16, 40, 128), (64, 24, 256), (64, 24, 512)])
def test_several_tokens_a_sequence(n1, batch, d):
    """Causal steps of three tokens, some sequences with fewer; own items of 32, 64 and 128 head rows, own tokens
    that span ranges; both modes."""
    prefix, tokens = 770, ([3, 1, 0, 2, 3] * 8)[:batch]
    kv = [prefix + v for v in ([3, 1, 40, 300, 2] * 8)[:batch]]
    t = make(BF, n1, d, [3] * batch, kv, prefix, 48, False, 510 + d)
    for mode in (0, 3):
        check(plan_of(t, tokens, kv, prefix, 0.04, mode).run(), exact(t, tokens, kv, prefix, 0.04, mode, False))


@pytest.mark.parametrize("width", WIDTHS)
def test_missing_blocks(width):
    n1, batch = WIDTHS[width]
    prefix = 1024
    kv = lengths(batch, prefix)
    t = make(BF, n1, 256, [1] * batch, kv, prefix, 16, False, 520)
    last = t["table"].shape[1] - 1
    t["table"][0, 0], t["table"][0, 7], t["table"][0, 63] = -1, t["k"].shape[0], 2 ** 31 - 1
    t["table"][4, 64], t["table"][1, 64] = -1, t["k"].shape[0] + 5
    t["table"][5, last] = -7
    check(plan_of(t, None, kv, prefix, 0.05).run(), exact(t, [1] * batch, kv, prefix, 0.05, 3, False))


@pytest.mark.parametrize("scale", [-0.04, 0.0, 0.4, -1.5])
@pytest.mark.parametrize("width", WIDTHS)
def test_scales(width, scale):
    n1, batch = WIDTHS[width]
    prefix = 900
    kv = lengths(batch, prefix)
    for dtype in (BF, HF):
        t = make(dtype, n1, 512, [1] * batch, kv, prefix, 32, False, 530)
        check(plan_of(t, None, kv, prefix, scale).run(), exact(t, [1] * batch, kv, prefix, scale, 3, False))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("width", WIDTHS)
def test_rising_scores(width, dtype):
    """Along the prefix each tile's maximum exceeds the one before by more than the lazy threshold."""
    n1, batch = WIDTHS[width]
    prefix, page = 800, 50
    kv = lengths(batch, prefix)
    t = make(dtype, n1, 512, [1] * batch, kv, prefix, page, False, 540)
    order = t["table"][0, :prefix // page].long()
    k = t["k"].view(-1, page, 512)
    k[order, :, 0] = torch.linspace(-150, 150, prefix).view(-1, page).to(dtype).cuda()
    t["q"][..., 0] = 4.0
    check(plan_of(t, None, kv, prefix, 0.9).run(), exact(t, [1] * batch, kv, prefix, 0.9, 3, False))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("width", WIDTHS)
def test_values_that_no_row_sees(width, value):
    """What is not finite in prefix tokens behind a short sequence's end, or behind the sequences, reaches only
    the rows that see it."""
    n1, batch = WIDTHS[width]
    prefix, page = 900, 32
    kv = lengths(batch, prefix)          # the last ends 37 tokens before the prefix, sequence 3 after 128
    t = make(BF, n1, 256, [1] * batch, kv, prefix, page, False, 550)
    want = exact(t, [1] * batch, kv, prefix, 0.04, 3, False)
    k, kr, tab = t["k"], t["kr"], t["table"].long()
    for b in range(batch):
        for p in range(max(kv[b], prefix), tab.shape[1] * page):
            k[tab[b, p // page], p % page] = value
            kr[tab[b, p // page], p % page] = value
    plan = plan_of(t, None, kv, prefix, 0.04)
    check(plan.run(), want)
    # the first prefix token behind the last sequence's end, in one column, and in the rotary part
    p = kv[-1]
    k[tab[0, p // page], p % page, 0, 7] = value
    kr[tab[0, p // page], p % page, 0, 3] = value
    got = plan.run()
    for b in (0, 3, batch - 1):
        check(got, want, rows=slice(b, b + 1))
    for b in set(range(batch)) - {0, 3, batch - 1}:
        assert torch.isnan(got[0][b, ..., 7]).all()
        if math.isnan(value):
            assert torch.isnan(got[0][b]).all()


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


@pytest.mark.parametrize("batch,n1,prefix,kv", [(4, 16, 32768, 32770), (2, 8, 13000, 13003), (1, 4, 0, 20000)])
def test_many_ranges(batch, n1, prefix, kv):
    """More ranges than the eight waves of the join take at first (12 each): its second loop."""
    kv = [kv + 70 * b for b in range(batch)]
    t = make(BF, n1, 512, [1] * batch, kv, prefix, 128, False, 580)
    plan = plan_of(t, None, kv, prefix, 0.04, least=97 if prefix else 0)
    assert sum(ranges(plan)) > 96
    check(plan.run(), exact(t, [1] * batch, kv, prefix, 0.04, 3, False))


@pytest.mark.parametrize("width", WIDTHS)
def test_plan_grows_far_past_its_lengths(width):
    """A captured run() of a plan built one token past the prefix, whose cut is of those lengths: 1500 tokens
    later the last own range has them all. Replays beside eager work."""
    n1, batch = WIDTHS[width]
    prefix, page = 1031, 64
    kv = [prefix + 1] * batch
    t = make(BF, n1, 512, [1] * batch, [v + 1600 for v in kv], prefix, page, False, 590)
    plan = plan_of(t, None, kv, prefix, 0.04)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    for step in (0, 1, 40, 1500):
        lens = [v + max(0, step - 7 * b) for b, v in enumerate(kv)]
        lens[2] = min(lens[2], prefix - 5)     # and one that ends inside the prefix now
        plan.act_k[:batch].copy_(torch.tensor(lens, dtype=torch.int32))
        t["q"].copy_(torch.randn_like(t["q"].float()).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        want = exact(t, [1] * batch, lens, prefix, 0.04, 3, False)
        check((plan.out, plan.sm[0], plan.sm[1]), want)
        eager = plan_of(t, None, lens, prefix, 0.04).run()
        check(eager, want)


@pytest.mark.parametrize("width", WIDTHS)
def test_runs_repeat_bit_for_bit(width):
    """No sum depends on the order in which work-groups run."""
    n1, batch = WIDTHS[width]
    prefix = 2000
    kv = lengths(batch, prefix)
    t = make(BF, n1, 512, [1] * batch, kv, prefix, 64, False, 600)
    plan = plan_of(t, None, kv, prefix, 0.04)
    first = [x.clone() for x in plan.run()]
    for _ in range(5):
        plan.ws.fill_(255)    # whatever the workspace held
        assert all(torch.equal(a, b) for a, b in zip(plan.run(), first))
