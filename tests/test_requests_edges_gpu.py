"""Adapters by request and their gradients at the edges of what the calls
promise: captured graphs, streams given, infinities, ranks below the bank's.

Tolerances are the bounds of test_requests_gpu.py, element by element.
"""
import contextlib

import numpy as np
import pytest
import torch

from mingproj._lib import MP_EINVAL, MP_ETIMEOUT
from mingproj.proj import Context, MP_QUANT_SYMMETRIC, MPError
from test_requests_gpu import ADD, BF, _bank, _bf16, _forward_ref, _grad_ref, _segments, _weight, _within

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


@pytest.mark.parametrize("m", [6, 260])
def test_calls_on_a_stream_given(ctx, m):
    """stream=: what a call converts is ordered on that stream, not on the busy
    current one, and its results take no memory that the current one still uses."""
    rng = np.random.default_rng(m)
    n, k, cap, r = 256, 128, 3, 16
    w, _, _ = _weight(ctx, rng, n, k, 8)
    wt = ctx.transposed(w)
    bank, fac = _bank(ctx, rng, n, k, cap, r, [r] * cap, training=True)
    plan = ctx.requests(3, m, cap)
    third = m // 3
    # int64, strided, a factor that is not contiguous: each is converted by the call
    lengths = torch.tensor([[third, 9], [third - 1, 9], [third, 9]], device="cuda")[:, 0]
    owners = torch.tensor([2, 0, 1], device="cuda")
    strengths = torch.tensor([1.0, 0.5, -2.0], dtype=torch.float64, device="cuda")
    a_t = fac[0][0].to(torch.bfloat16).T.contiguous().T
    b_t = fac[0][1].to(torch.bfloat16).T.contiguous().T
    x, dy = _bf16(rng, m, k), _bf16(rng, m, n)

    def step(stream=None):
        bank.set(1, a_t, b_t, stream=stream)
        plan.plan(lengths, owners, strengths, m, stream=stream)
        y, v = ctx.linear_requests(w, x, bank, plan, ranks=True, stream=stream)
        saved = ctx.checkpoint(x, stream=stream)
        back = ctx.restore(saved, stream=stream)
        return (y, v, saved.codes, saved.scales, back) + ctx.linear_requests_grad(wt, dy, saved, v, bank, plan,
                                                                                 stream=stream)

    want = step()
    torch.cuda.synchronize()
    # another plan and factor in place, so that a stale conversion would show
    bank.set(1, -a_t, b_t)
    plan.plan([m], [1], None, m)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    for _ in range(3):
        # memory given back whose last use on the current stream is still to come
        old = [torch.empty_like(t) for t in want for _ in range(2)]
        for _ in range(20):
            busy @ busy
        for t in old:
            t.fill_(7)
        del old, t
        got = step(stream=side)
        side.synchronize()
        kept = [t.clone() for t in got]
        torch.cuda.synchronize()
        for p, q, s in zip(want, kept, got):
            assert torch.equal(p, q) and torch.equal(p, s)
    ctx.sync_check()
    for h in (w, wt, bank, plan):
        h.free()


def _like(got, ref, name):
    """Infinities and NaN where the formula in 64 bits has them, with its signs."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{name}: NaN in other places"
    wild = torch.isinf(ref)
    assert torch.equal(torch.isinf(got), wild) and torch.equal(got[wild], ref[wild]), f"{name}: other infinities"


# rank-space rows in runs; runs, then the projection; the tensor core's tiles with and without a cluster
@pytest.mark.parametrize("m,k,bits", [(6, 640, 0), (90, 640, 8), (2100, 640, 0), (3000, 128, 4)])
def test_infinite_rows_and_ranks_below_the_banks(ctx, m, k, bits):
    """An infinity in x meets an adapter's own ranks and not the padding up to the
    bank's; an adapter that was never set adds nothing to it."""
    rng = np.random.default_rng(m + k)
    n, cap, ranks = 256, 3, [3, 20]
    w, w64, _ = _weight(ctx, rng, n, k, bits)
    bank, fac = _bank(ctx, rng, n, k, cap, 20, ranks)  # adapter 2: never set
    plan = ctx.requests(3, m, cap)
    q = m // 3
    x = _bf16(rng, m, k)
    rows = [0, q - 1, q, 2 * q, m - 1]
    for i, t in enumerate(rows):
        x[t, (17 * i + 5) % k] = float("inf") * (-1) ** i
    plan.plan([q, q, m - 2 * q], [0, 1, 2], [0.5, -1.0, 1.0], m)
    y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
    plan.plan([q, q, m - 2 * q], [0, 1, -1], [0.5, -1.0, 1.0], m)
    y0, v0 = ctx.linear_requests(w, x, bank, plan, ranks=True)
    ctx.sync_check()
    assert torch.equal(y[2 * q:].view(torch.int16), y0[2 * q:].view(torch.int16)), "never set: the base's bits"
    assert not v[:q, 3:].any() and not v[:, 20:].any() and not v[2 * q:].any() and not v0[2 * q:].any()
    rv = torch.zeros(m, bank.rank_pad, dtype=torch.float64, device="cuda")
    ry = x.double() @ w64.T
    for at, a, s in ((slice(0, q), 0, 0.5), (slice(q, 2 * q), 1, -1.0)):
        t = s * (x[at].double() @ fac[a][0].T)
        rv[at, :ranks[a]] = t
        ry[at] += t @ fac[a][1].T
    assert torch.isinf(ry).any()
    _like(v, rv, "v")
    _like(y, ry, "y")
    for h in (w, bank, plan):
        h.free()


@pytest.mark.parametrize("bits,mode", [(0, 0), (8, 0), (4, 0), (8, MP_QUANT_SYMMETRIC)])
@pytest.mark.parametrize("m", [1, 6, 16, 32, 33])
def test_wild_rows_of_few(ctx, m, bits, mode):
    """Up to 32 rows the codes of a packed weight are multiplied as whole numbers:
    infinities, and values whose products with the codes overflow where those
    with the weights do not, come out as the formula has them."""
    rng = np.random.default_rng(m + bits)
    n, k, cap, r = 264, 320, 2, 16
    w, w64, wround = _weight(ctx, rng, n, k, bits, mode)
    bank, fac = _bank(ctx, rng, n, k, cap, r, [r, 5])
    lengths, owners, strengths = [m - m // 2, m // 4], [1, 0], [0.5, -1.0]
    plan = ctx.requests(2, m, cap)
    plan.plan(lengths, owners, strengths, m)
    segs = list(_segments(m, lengths, owners, strengths))
    for value in (float("inf"), float("-inf"), float("nan"), 3e37, -1e38):
        x = _bf16(rng, m, k)
        for t in range(0, m, 2):
            x[t, (7 * t + 64) % k] = value
        y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
        ctx.sync_check()
        ry, by, rv, bv = _forward_ref(x, w64, wround, fac, segs, bank.rank_pad)
        # (the bound's NaN and infinities stand where the formula's are)
        fine = torch.isfinite(ry)
        assert fine.all() or not np.isfinite(value)
        if not np.isfinite(value):
            _like(y, ry, "y")
        zero = torch.zeros_like(ry)
        _within("y", torch.where(fine, y.double(), zero), torch.where(fine, ry, zero), torch.where(fine, by, zero + 1))
        if np.isfinite(value):
            _within("v", v, rv, bv)
    for h in (w, bank, plan):
        h.free()


# m, n, k, capacity, bank's rank, rows of the requests (adapter 0, 1, 0): clusters and walking CTAs, every width of sums
WILD_GRADS = [
    (33, 136, 200, 2, 7, [11, 10, 9]),
    (700, 264, 640, 3, 16, [300, 100, 299]),
    (1500, 1280, 1024, 40, 12, [500, 480, 510]),
    (900, 640, 520, 2, 64, [300, 300, 300]),
    (1200, 1280, 1024, 24, 50, [400, 380, 410]),
    (640, 512, 392, 2, 128, [200, 200, 200]),
    (700, 1280, 1280, 16, 100, [230, 210, 240]),
]


@pytest.mark.parametrize("saved", [16, 8])
@pytest.mark.parametrize("case", WILD_GRADS, ids=[f"m{c[0]}_cap{c[3]}_r{c[4]}" for c in WILD_GRADS])
def test_wild_values_in_gradients(ctx, case, saved):
    """u and v are multiplied in three parts: an infinity in x or dy meets what
    they are and not their parts; a checkpoint's scale that overflows with u does
    not reach the codes that are 0."""
    m, n, k, cap, max_rank, lengths = case
    rng = np.random.default_rng(m + max_rank + saved)
    ranks = [max_rank, max(1, max_rank // 3)]
    owners, strengths = [0, 1, 0], [1.0, -0.5, 0.75]
    w, w64, wround = _weight(ctx, rng, n, k, 0)
    wt = ctx.transposed(w)
    bank, fac = _bank(ctx, rng, n, k, cap, max_rank, ranks, training=True)
    plan = ctx.requests(3, m, cap)
    plan.plan(lengths, owners, strengths, m)
    segs = list(_segments(m, lengths, owners, strengths))
    rows = [0, lengths[0] + 1, lengths[0] + lengths[1] + 2, sum(lengths) - 1]
    for which, value in (("x", float("inf")), ("dy", float("-inf")), ("x", float("nan")), ("x", 3e38)):
        x, dy = _bf16(rng, m, k), _bf16(rng, m, n)
        for i, t in enumerate(rows):
            (x if which == "x" else dy)[t, 3 + 131 * (i % 2)] = value * (-1) ** i
        if value == 3e38:
            dy *= 64.0  # u past 1 / 2.4e36 of f32's largest
        _, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
        v = torch.where(torch.isfinite(v), v, torch.zeros_like(v)) if which == "x" else v
        x_in = ctx.checkpoint(x) if saved == 8 else x
        kept = x if saved == 16 else x_in.codes.double() * x_in.scales.double().repeat_interleave(128, 1)[:, :k]
        dx, da, db = ctx.linear_requests_grad(wt, dy, x_in, v, bank, plan)
        again = ctx.linear_requests_grad(wt, dy, x_in, v, bank, plan)
        ctx.sync_check()
        refs = _grad_ref(kept, dy, w64, wround, fac, segs, v, cap, max_rank)
        for a, r in enumerate(ranks):  # a product with the padding is none
            refs[2][0][a, :, r:] = 0.0
            refs[2][1][a, :, r:] = 1e-30
        for name, got, twice, (ref, bound) in zip(("dx", "da", "db"), (dx, da, db), again, refs):
            assert torch.equal(got.view(torch.int16), twice.view(torch.int16)), "the same call twice"
            if value != 3e38:
                _like(got, ref, name)
            # where the sum of the products' magnitudes (at most 2^16 of the bound) fits f32
            fine = torch.isfinite(ref) & (bound < 2.0 ** -16 * 1e38)
            assert fine.any()
            zero = torch.zeros_like(ref)
            _within(name, torch.where(fine, got.double(), zero), torch.where(fine, ref, zero),
                    torch.where(fine, bound, zero + 1))
    for h in (w, wt, bank, plan):
        h.free()


# shapes whose K splits differ between the whole call's rows, a quarter and a sixteenth
@pytest.mark.parametrize("m,n,k", [(2048, 512, 3840), (1024, 1024, 2560)])
def test_image_rows_do_not_enter(ctx, m, n, k):
    """Kernel, tile and splits of a call with adapters by request come from the
    whole call: a count of rows an image, or row segments, set for other launches
    change no bit."""
    rng = np.random.default_rng(m)
    cap, r = 2, 16
    w, _, _ = _weight(ctx, rng, n, k, 8)
    bank, _ = _bank(ctx, rng, n, k, cap, r, [r, r])
    plan = ctx.requests(2, m, cap)
    plan.plan([m // 2, m // 2], [0, 1], None, m)
    x = _bf16(rng, m, k)
    want = ctx.linear_requests(w, x, bank, plan)
    try:
        ctx.set_image_rows(m // 16)
        by_images = ctx.linear_requests(w, x, bank, plan)
        ctx.set_image_rows(0)
        ctx.set_strengths_rows(np.ones((4, 8), np.float32), [i * m // 4 for i in range(5)])
        by_segments = ctx.linear_requests(w, x, bank, plan)
    finally:
        ctx.set_image_rows(0)
        ctx.clear_strengths_rows()
    ctx.sync_check()
    assert torch.equal(want, by_images) and torch.equal(want, by_segments)
    for h in (w, bank, plan):
        h.free()


def test_a_cut_plan_is_reported_beside_a_timeout(ctx):
    plan = ctx.requests(1, 8, 1)
    for timeout in (True, False):
        plan.plan([9], [0], None, 8)  # a row too many
        if timeout:
            ctx.selftest_wait(1_000_000)  # 1 ms
            with pytest.raises(MPError) as e:
                ctx.sync_check()
            assert e.value.status == MP_ETIMEOUT
        with pytest.raises(MPError, match="out of range") as e:
            ctx.sync_check()
        assert e.value.status == MP_EINVAL
        ctx.sync_check()
    plan.free()


@contextlib.contextmanager
def _refusing_stream():
    """A stream whose capture was broken off: every launch on it fails on the host."""
    from cuda.bindings import runtime
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    relaxed = runtime.cudaStreamCaptureMode.cudaStreamCaptureModeRelaxed
    assert runtime.cudaStreamBeginCapture(side.cuda_stream, relaxed)[0] == runtime.cudaError_t.cudaSuccess
    assert runtime.cudaStreamSynchronize(side.cuda_stream)[0] != runtime.cudaError_t.cudaSuccess  # not allowed there
    try:
        with torch.cuda.stream(side):
            yield
    finally:
        assert runtime.cudaStreamEndCapture(side.cuda_stream)[0] != runtime.cudaError_t.cudaSuccess


def test_a_failed_launch_fails_one_call(ctx):
    """The call after a failed one does not report its error again."""
    rng = np.random.default_rng(1)
    n, k = 128, 64
    bank, fac = _bank(ctx, rng, n, k, 1, 8, [8])
    plan = ctx.requests(4, 40, 1)
    lengths, owners = (torch.tensor([v] * 4, dtype=torch.int32, device="cuda") for v in (10, 0))
    with _refusing_stream(), pytest.raises(MPError):
        plan.plan(lengths, owners, None, 40)
    bank.set(0, *(f.to(torch.bfloat16) for f in fac[0]))
    ctx.sync_check()
    for h in (bank, plan):
        h.free()


def test_a_plan_that_fails_leaves_the_one_before(ctx):
    """Calls of the rows planned before still run, calls of the new ones are refused."""
    rng = np.random.default_rng(2)
    m, n, k = 40, 128, 64
    w, _, _ = _weight(ctx, rng, n, k, 8)
    bank, _ = _bank(ctx, rng, n, k, 1, 8, [8])
    plan = ctx.requests(4, 4 * m, 1)
    x = _bf16(rng, 4 * m, k)
    lengths, owners = (torch.tensor([v] * 4, dtype=torch.int32, device="cuda") for v in (m, 0))
    plan.plan([m], [0])
    want = ctx.linear_requests(w, x[:m], bank, plan)
    with _refusing_stream(), pytest.raises(MPError):
        plan.plan(lengths, owners, None, 4 * m)
    with pytest.raises(MPError, match="rows were planned"):
        ctx.linear_requests(w, x, bank, plan)
    assert torch.equal(ctx.linear_requests(w, x[:m], bank, plan), want)
    ctx.sync_check()
    for h in (w, bank, plan):
        h.free()


@pytest.mark.parametrize("bits,mode", [(8, 0), (4, 0), (8, MP_QUANT_SYMMETRIC)])
def test_transposed_weight_and_few_rows(ctx, bits, mode):
    """Up to 32 rows the forward weight is the codes' own, scale and bias in f32;
    the transpose holds it rounded to bf16. Unit rows show both: each within one
    rounding of the weight, so within two of one another."""
    rng = np.random.default_rng(bits + mode)
    n, k, top = 192, 128, 2 ** bits
    w, w64, _ = _weight(ctx, rng, n, k, bits, mode)
    wt = ctx.transposed(w)
    bank, _ = _bank(ctx, rng, n, k, 1, 8, [8])
    plan = ctx.requests(1, 33, 1)
    rows = torch.eye(k, dtype=torch.bfloat16, device="cuda").repeat(2, 1)  # whole calls of 33 rows
    back = ctx.linear(wt, torch.eye(n, dtype=torch.bfloat16, device="cuda"))  # [n, k]
    # sums of scale * code and bias in f32 may cancel: codes reach 2^bits, or 128 + 2^4, steps
    step = (w64.max(1).values - w64.min(1).values)[:, None] / (top - 1) * 1.5
    near = 4 * ADD * step * max(top, 144)
    for m in (32, 33):
        plan.plan([], [], None, m)
        few = torch.cat([ctx.linear_requests(w, rows[i:i + m], bank, plan).T for i in range(0, k, m)], 1)[:, :k]
        ctx.sync_check()
        if m == 33:
            assert torch.equal(few, back), "above 32 rows: the same bf16 weight"
        rounding = BF * w64.abs() * (1 + BF) + near
        assert ((few.double() - w64).abs() <= rounding).all()
        assert ((few.double() - back.double()).abs() <= 2 * rounding).all()
    for h in (w, wt, bank, plan):
        h.free()
