"""Adapters by request and their gradients at the edges of what the calls
promise: captured graphs, streams given, infinities, ranks below the bank's.

Tolerances are the bounds of test_requests_gpu.py, element by element.
"""
import numpy as np
import pytest
import torch

from mingproj.proj import Context
from test_requests_gpu import _bank, _bf16, _weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,larger", [(6, 30), (90, 2100)])
def test_graph_outlives_larger_calls(m, larger):
    """A buffer that grows after a capture stays: a replay gives the capture's
    bits although a larger call came between and freed memory was written."""
    rng = np.random.default_rng(m)
    ctx = Context(torch.cuda.current_device())  # nothing captured in it before
    n, k = 512, 640
    w, _, _ = _weight(ctx, rng, n, k, 8)
    wt = ctx.transposed(w)
    small, _ = _bank(ctx, rng, n, k, 2, 16, [16, 8], training=True)
    large, _ = _bank(ctx, rng, n, k, 2, 128, [128, 100], training=True)

    def step(bank, plan, x, dy):
        y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
        z = ctx.linear_requests(w, x, bank, plan)  # its rank-space rows in the context's memory
        return (y, z) + ctx.linear_requests_grad(wt, dy, x, v, bank, plan)

    def batch(rows):
        plan = ctx.requests(2, rows, 2)
        plan.plan([rows // 2, rows // 3], [0, 1], None, rows)
        return plan, _bf16(rng, rows, k), _bf16(rng, rows, n)

    a, b = batch(m), batch(larger)
    want = step(small, *a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(small, *a)
    graph.replay()
    torch.cuda.synchronize()
    step(large, *b)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    junk = [torch.full((1 << s,), float("nan"), device="cuda") for s in range(8, 24) for _ in range(2)]
    for t in outs:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, outs))
    assert all(torch.isnan(t).all() for t in junk), "a replay wrote into freed memory"
    ctx.sync_check()
    del graph
    for h in (a[0], b[0], small, large, wt, w):
        h.free()
    ctx.close()
