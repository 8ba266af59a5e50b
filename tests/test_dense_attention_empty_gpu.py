"""Plans of dense_attention and its gradient without a row or a key: each run clears the outputs, on its own stream."""
import pytest
import torch

import dsa_triton_ascend_amd as dsa

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SHAPES = [("TND", (5, 4, 64), (0, 2, 64)), ("BSND", (2, 5, 4, 64), (2, 0, 2, 64)), ("TND", (0, 4, 64), (7, 2, 64))]


def plans(layout, qs, ks):
    q, k = torch.ones(qs, dtype=BF, device="cuda"), torch.ones(ks, dtype=BF, device="cuda")
    fwd = dsa.DenseAttentionPlan(q, k, k, layout=layout, return_softmax_lse=True)
    out, mx, sm = fwd.run()
    return [fwd, dsa.DenseAttentionGradPlan(q, k, k, q, out, mx, sm, layout=layout)]


@pytest.mark.parametrize("layout,qs,ks", SHAPES)
@pytest.mark.parametrize("captured", [False, True])
def test_each_run_clears(layout, qs, ks, captured):
    for plan in plans(layout, qs, ks):
        first = [x for x in plan.run() if x is not None]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                plan.run()
        for _ in range(3):
            for x in first:
                x.fill_(3.0)
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                if captured:
                    graph.replay()
                else:
                    again = [x for x in plan.run() if x is not None]
                    assert all(a is b for a, b in zip(first, again))
                assert not any(bool(x.any()) for x in first)
            torch.cuda.current_stream().wait_stream(s)


@pytest.mark.parametrize("layout,qs,ks", SHAPES)
def test_in_place_when_the_constructor_returns(layout, qs, ks):
    """What a plan made behind much work on its stream returns is whole on another stream that waits for nothing"""
    x = torch.randn(8192, 8192, device="cuda")
    for at in (0, 1):
        torch.cuda.synchronize()
        for _ in range(20):
            x = x @ x
        plan = plans(layout, qs, ks)[at]
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs = [o.clone() for o in plan.run() if o is not None]
        s.synchronize()
        assert not any(bool(o.any()) for o in outs)
