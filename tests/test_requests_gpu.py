"""Adapters by request (mp_linear_requests, its backward pass) and 8-bit
activation checkpoints against plain 64-bit arithmetic.

Tolerances are bounds, element by element, from the roundings the kernels make:
  y   bf16 output (2^-8 |y|), bf16 weight after dequantization (2^-8 sum |x||W|,
      packed weights only), bf16 rank-space rows (2^-8 sum |v||B|), and f32
      sums, which lose at most 2^-23 of the sum of magnitudes per term added
  v   f32 sums alone
  dx  as y, with W, v, B read as W^T, u, A
  dA, dB  f32 sums, and factors of the products kept to 2^-16 or better
"""
import math

import numpy as np
import pytest
import torch

from mingproj import pack as P
from mingproj.proj import Checkpoint, Context, MPError, MP_QUANT_SYMMETRIC

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8   # bf16 rounding, relative (8 significant bits: half a unit in the last place)
ADD = 2.0 ** -23  # one f32 addition


def _bf16(rng, *shape, scale=1.0):
    return torch.from_numpy(rng.normal(size=shape).astype(np.float32) * scale).to(torch.bfloat16).cuda()


def _weight(ctx, rng, n, k, bits, mode=0):
    """(handle, W in f64 on the device, rounding of W)."""
    if bits == 0:
        w = _bf16(rng, n, k, scale=1 / math.sqrt(k))
        return ctx.upload(n, k, 0, w), w.double(), 0.0
    pw = P.synthetic_symmetric_w8(rng, n, k) if mode == MP_QUANT_SYMMETRIC else P.synthetic_affine(rng, n, k, bits)
    h = ctx.upload(n, k, bits, pw.data, pw.scales, pw.biases, mode=pw.mode)
    per = 32 // bits
    words = torch.from_numpy(pw.data.astype(np.int64)).reshape(n, -1)
    q = (words[:, :, None] >> (bits * torch.arange(per))) & (2 ** bits - 1)
    q = q.reshape(n, k).double()
    if mode == MP_QUANT_SYMMETRIC:
        q = torch.where(q > 127, q - 256, q)
    up = lambda b: torch.from_numpy(P.bf16_bits_to_f32(b)).double().repeat_interleave(64, 1)  # noqa: E731
    w = q * up(pw.scales) + (up(pw.biases) if pw.biases is not None else 0.0)
    return h, w.cuda(), BF


def _bank(ctx, rng, n, k, cap, max_rank, ranks, training=False):
    bank = ctx.adapters(n, k, cap, max_rank, training=training)
    fac = []
    for i, r in enumerate(ranks):
        a, b = _bf16(rng, r, k, scale=1 / math.sqrt(k)), _bf16(rng, n, r, scale=0.5 / math.sqrt(r))
        bank.set(i, a, b)
        fac.append((a.double(), b.double()))
    return bank, fac


def _segments(m, lengths, adapters, strengths):
    at = 0
    for n, a, s in zip(lengths, adapters, strengths):
        lo, hi = min(at, m), min(at + n, m)
        at += n
        if a >= 0 and hi > lo and s != 0.0:
            yield slice(lo, hi), a, s


def _forward_ref(x, w, wround, fac, segs, rank_pad):
    """(y, bound on |error|, v, its bound) in f64."""
    m, k = x.shape
    x = x.double()
    y = x @ w.T
    mag = x.abs() @ w.abs().T
    err = wround * mag
    v = torch.zeros(m, rank_pad, dtype=torch.float64, device=x.device)
    verr = torch.zeros_like(v)
    terms = k
    for rows, a, s in segs:
        fa, fb = fac[a]
        r = fa.shape[0]
        t = s * (x[rows] @ fa.T)
        te = (k + 2) * ADD * abs(s) * (x[rows].abs() @ fa.abs().T)
        v[rows, :r], verr[rows, :r] = t, te
        y[rows] += t @ fb.T
        low = t.abs() @ fb.abs().T
        err[rows] += BF * low + te @ fb.abs().T
        mag[rows] += low
        terms = k + 128
    err += terms * ADD * mag
    return y, err * (1 + 4 * BF) + BF * y.abs() + 1e-30, v, verr + 1e-30


def _within(name, got, ref, bound):
    off = (got.double() - ref).abs()
    worst = (off / bound).max().item()
    assert torch.isfinite(got.double()).all() and worst <= 1.0, f"{name}: {worst:.3g} of the bound"


CASES = [
    # m, n, k, cap, max rank, lengths, adapters, strengths
    (1, 128, 64, 1, 1, [1], [0], [1.0]),
    (1, 384, 640, 3, 16, [1], [2], [-0.7]),
    (7, 256, 128, 4, 12, [1, 0, 2, 1, 3], [3, 1, -1, 0, 3], [1.0, 1.0, 1.0, 0.5, -1.0]),
    (16, 640, 512, 16, 32, [1] * 16, list(range(15, -1, -1)), [0.5 + 0.1 * i for i in range(16)]),
    (33, 264, 192, 2, 40, [0, 33, 0], [0, 1, 0], [1.0, 0.3, 1.0]),
    (64, 128, 320, 5, 64, [8] * 8, [0, 1, 2, 3, 4, 0, -1, 2], [1.0] * 8),
    (130, 136, 192, 3, 17, [63, 1, 64], [2, 0, 1], [1.0, 2.0, -1.0]),  # ends inside and on a tile
    (200, 192, 128, 7, 16, [1] * 200, [(3 * i) % 8 - 1 for i in range(200)], [1.0] * 200),  # a token each
    (300, 256, 256, 4, 128, [129, 5, 100], [3, 0, 3], [0.2, 1.0, 1.0]),  # one adapter twice, rows left over
    (517, 648, 640, 6, 24, [50, 51, 0, 200, 3, 1, 212], [5, 4, 3, 2, 1, -1, 0], [1, 1, 1, 0.0, 1, 1, 1.5]),
    (1100, 512, 512, 2, 80, [600, 500], [1, 0], [1.0, 1.0]),
]


@pytest.mark.parametrize("bits,mode", [(0, 0), (8, 0), (4, 0), (8, MP_QUANT_SYMMETRIC)])
@pytest.mark.parametrize("case", CASES, ids=[f"m{c[0]}_n{c[1]}_k{c[2]}_r{c[4]}" for c in CASES])
def test_linear_requests(ctx, bits, mode, case):
    m, n, k, cap, max_rank, lengths, adapters, strengths = case
    rng = np.random.default_rng(m + n + bits)
    w, w64, wround = _weight(ctx, rng, n, k, bits, mode)
    ranks = [max(1, max_rank >> (i % 3)) for i in range(cap)]
    bank, fac = _bank(ctx, rng, n, k, cap, max_rank, ranks)
    plan = ctx.requests(len(lengths), m, cap)
    plan.plan(lengths, adapters, strengths, m)
    x = _bf16(rng, m, k)
    out = torch.full((m, (n + 7) // 8 * 8), float("nan"), dtype=torch.bfloat16, device="cuda")[:, :n]
    y, v = ctx.linear_requests(w, x, bank, plan, out=out, ranks=True)
    again = ctx.linear_requests(w, x, bank, plan)
    ctx.sync_check()
    ry, by, rv, bv = _forward_ref(x, w64, wround, fac, list(_segments(m, lengths, adapters, strengths)),
                                  bank.rank_pad)
    _within("y", y, ry, by)
    _within("v", v, rv, bv)
    assert torch.equal(y, again), "the same call twice"
    for h in (w, bank, plan):
        h.free()


LONG = [
    # enough to multiply for the tensor-core kernels, K split in clusters and not;
    # long runs of rows for one adapter (the sums of dA and dB)
    (2100, 384, 640, 3, 128, [1500, 1, 0, 590], [1, 0, 2, 1], [1.0, 1.0, 1.0, -0.5]),
    (5000, 264, 1032, 2, 20, [4990], [1], [0.7]),
    (4100, 1024, 768, 12, 64, [300, 257, 511, 64, 1, 900, 128, 640, 777, 33, 400], list(range(11)), [1.0] * 11),
    (700, 256, 3328, 5, 48, [100, 128, 130, 12, 330], [0, 1, 4, 2, 3], [1.0, -1.0, 0.25, 1.0, 0.0]),
]


@pytest.mark.parametrize("case", LONG, ids=[f"m{c[0]}_n{c[1]}_k{c[2]}_r{c[4]}" for c in LONG])
@pytest.mark.parametrize("saved", [16, 8])
def test_long_requests(ctx, case, saved):
    m, n, k, cap, max_rank, lengths, adapters, strengths = case
    rng = np.random.default_rng(3 * m + n + saved)
    w, w64, wround = _weight(ctx, rng, n, k, 0)
    bank, fac = _bank(ctx, rng, n, k, cap, max_rank, [max(1, max_rank - 3 * i) for i in range(cap)], training=True)
    plan = ctx.requests(len(lengths), m, cap)
    plan.plan(lengths, adapters, strengths, m)
    x, dy = _bf16(rng, m, k), _bf16(rng, m, n, scale=0.1)
    segs = list(_segments(m, lengths, adapters, strengths))
    y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
    wt = ctx.transposed(w)
    x_in = ctx.checkpoint(x) if saved == 8 else x
    kept = x if saved == 16 else x_in.codes.double() * x_in.scales.double().repeat_interleave(128, 1)[:, :k]
    dx, da, db = ctx.linear_requests_grad(wt, dy, x_in, v, bank, plan)
    again = ctx.linear_requests_grad(wt, dy, x_in, v, bank, plan)
    ctx.sync_check()
    ry, by, rv, bv = _forward_ref(x, w64, wround, fac, segs, bank.rank_pad)
    _within("y", y, ry, by)
    _within("v", v, rv, bv)
    rx, ra, rb = _grad_ref(kept, dy, w64, wround, fac, segs, v, cap, max_rank)
    _within("dx", dx, *rx)
    _within("da", da, *ra)
    _within("db", db, *rb)
    for name, got, ref in (("v", v, rv), ("da", da, ra[0]), ("db", db, rb[0])):
        # as near as sums in f32 with rounding to nearest come at these lengths:
        # 2^-24 of the result a term, added at random, and 2^-17 of a factor
        off = ((got.double() - ref).norm() / ref.norm()).item()
        assert off <= 2.0 ** -24 * math.sqrt(m + n + k) + 2.0 ** -17, f"{name}: {off:.3g}"
    assert all(torch.equal(a, b) for a, b in zip((dx, da, db), again)), "the same call twice"
    for h in (w, wt, bank, plan):
        h.free()


NARROW = [
    # many rows of few features: little to multiply, the tensor core's tiles all the same
    (9000, 136, 64, 3, 64, [4100, 3, 64, 63, 4600], [2, 0, 1, -1, 0], [1.0, 0.5, 1.0, 1.0, -1.0]),
    (3000, 64, 192, 1, 16, [1500, 1500], [0, 0], [1.0, 0.25]),
    (2048, 72, 128, 4, 100, [16] * 128, [(3 * i) % 5 - 1 for i in range(128)], [1.0] * 128),
    (2500, 320, 256, 8, 40, [17] * 147, [(3 * i) % 9 - 1 for i in range(147)], [0.5 + i / 100 for i in range(147)]),
]


@pytest.mark.parametrize("case", NARROW, ids=[f"m{c[0]}_n{c[1]}_k{c[2]}_r{c[4]}" for c in NARROW])
@pytest.mark.parametrize("saved", [16, 8])
def test_narrow_long_requests(ctx, case, saved):
    test_long_requests(ctx, case, saved)


@pytest.mark.parametrize("rank,saved", [(4, 8), (4, 16), (30, 16), (64, 8), (100, 16)])
def test_gradients_repeat(ctx, rank, saved):
    """Hundreds of passes in a row, nothing waited for between them: the same
    bits every time, and no bounded wait given up."""
    rng = np.random.default_rng(rank)
    m, n, k, cap = 3000, 640, 896, 3
    w, _, _ = _weight(ctx, rng, n, k, 0)
    bank, _ = _bank(ctx, rng, n, k, cap, rank, [rank] * cap, training=True)
    plan = ctx.requests(4, m, cap)
    plan.plan([1300, 77, 900, 650], [0, 2, 2, 0], None, m)
    x, dy = _bf16(rng, m, k), _bf16(rng, m, n)
    wt = ctx.transposed(w)
    _, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
    x_in = ctx.checkpoint(x) if saved == 8 else x
    first = ctx.linear_requests_grad(wt, dy, x_in, v, bank, plan)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(300):
        for a, b in zip(first, ctx.linear_requests_grad(wt, dy, x_in, v, bank, plan)):
            differ += (a != b).sum()
    ctx.sync_check()
    assert int(differ) == 0
    for h in (w, wt, bank, plan):
        h.free()


def test_dense_any_k(ctx):
    """A dense weight with k not a multiple of 8, x's rows strided, NaN beside them."""
    rng = np.random.default_rng(5)
    m, n, k = 37, 130, 100 + 3
    w, w64, wround = _weight(ctx, rng, n, k, 0)
    bank, fac = _bank(ctx, rng, n, k, 2, 9, [9, 4])
    plan = ctx.requests(3, m, 2)
    lengths, adapters, strengths = [20, 10, 5], [0, 1, 0], [1.0, -2.0, 0.25]
    plan.plan(lengths, adapters, strengths, m)
    wide = torch.full((m, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = wide[:, :k]
    x.copy_(_bf16(rng, m, k))
    y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
    ctx.sync_check()
    ry, by, rv, bv = _forward_ref(x, w64, wround, fac, list(_segments(m, lengths, adapters, strengths)), bank.rank_pad)
    _within("y", y, ry, by)
    _within("v", v, rv, bv)
    for h in (w, bank, plan):
        h.free()


@pytest.mark.parametrize("m", [5, 70, 700])
def test_rows_without_adapter_have_the_base_bits(ctx, m):
    """No adapter, strength 0, an empty request and rows past the last request:
    the bits of the same call with an empty plan."""
    rng = np.random.default_rng(m)
    n, k = 256, 256
    w, _, _ = _weight(ctx, rng, n, k, 8)
    bank, _ = _bank(ctx, rng, n, k, 2, 16, [16, 8])
    plan = ctx.requests(4, m, 2)
    x = _bf16(rng, m, k)
    plan.plan([], [], None, m)
    base = ctx.linear_requests(w, x, bank, plan)
    q = m // 5
    plan.plan([q, q, 0, q], [0, -1, 1, 1], [1.0, 1.0, 1.0, 0.0], m)
    y = ctx.linear_requests(w, x, bank, plan)
    ctx.sync_check()
    assert torch.equal(y[q:], base[q:])
    assert not torch.equal(y[:q], base[:q])
    for h in (w, bank, plan):
        h.free()


@pytest.mark.parametrize("m,lengths", [(12, [4, 4, 4]), (150, [60, 30, 60]), (900, [300, 300, 300])])
def test_requests_do_not_touch_one_another(ctx, m, lengths):
    """An infinity or NaN in one request's rows or adapter stays there."""
    rng = np.random.default_rng(m)
    n, k = 256, 192
    w, _, _ = _weight(ctx, rng, n, k, 4)
    bank, fac = _bank(ctx, rng, n, k, 3, 16, [16, 16, 16], training=True)
    plan = ctx.requests(3, m, 3)
    plan.plan(lengths, [0, 1, 2], None, m)
    x, dy = _bf16(rng, m, k), _bf16(rng, m, n)
    y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
    wt = ctx.transposed(w)
    dx, da, db = ctx.linear_requests_grad(wt, dy, x, v, bank, plan)
    lo, hi = lengths[0], lengths[0] + lengths[1]
    others = [i for i in range(m) if not lo <= i < hi]

    x2, dy2 = x.clone(), dy.clone()
    x2[lo, 3], x2[hi - 1, 5] = float("nan"), float("inf")
    dy2[lo, 7], dy2[hi - 1, 9] = float("-inf"), float("nan")
    y2, v2 = ctx.linear_requests(w, x2, bank, plan, ranks=True)
    dx2, da2, db2 = ctx.linear_requests_grad(wt, dy2, x2, v2, bank, plan)
    assert torch.equal(y[others], y2[others]) and torch.equal(dx[others], dx2[others])
    assert not torch.isfinite(y2[lo]).any() and not torch.isfinite(dx2[lo]).any()
    for i in (0, 2):
        assert torch.equal(da[i], da2[i]) and torch.equal(db[i], db2[i])
    assert not torch.isfinite(da2[1]).all() and not torch.isfinite(db2[1]).all()

    a, b = (f.to(torch.bfloat16) for f in fac[1])
    for bad_a, bad_b in ((None, (17, 3)), ((2, 11), None)):
        a2, b2 = a.clone(), b.clone()
        if bad_a is not None:
            a2[bad_a] = float("inf")
        if bad_b is not None:
            b2[bad_b] = float("nan")
        bank.set(1, a2, b2)
        y3 = ctx.linear_requests(w, x, bank, plan)
        dx3, da3, db3 = ctx.linear_requests_grad(wt, dy, x, v, bank, plan)
        assert torch.equal(y[others], y3[others]) and torch.equal(dx[others], dx3[others])
        assert torch.isnan(y3[lo:hi]).all() and torch.isnan(dx3[lo:hi]).all()
        assert torch.equal(da[0], da3[0]) and torch.equal(da[2], da3[2])
    bank.set(1, a, b)  # set again: as before
    assert torch.equal(ctx.linear_requests(w, x, bank, plan), y)
    ctx.sync_check()
    for h in (w, wt, bank, plan):
        h.free()


def test_plan_cuts_what_is_out_of_range(ctx):
    rng = np.random.default_rng(3)
    m, n, k = 40, 128, 64
    w, w64, wround = _weight(ctx, rng, n, k, 0)
    bank, fac = _bank(ctx, rng, n, k, 2, 8, [8, 8])
    plan = ctx.requests(4, m, 2)
    x = _bf16(rng, m, k)
    for lengths, adapters, segs in (
            ([10, -3, 10], [0, 1, 1], [(slice(0, 10), 0, 1.0), (slice(10, 20), 1, 1.0)]),
            ([10, 100, 10], [0, 1, 0], [(slice(0, 10), 0, 1.0), (slice(10, 40), 1, 1.0)]),
            ([10, 10], [2, 1], [(slice(10, 20), 1, 1.0)]),
            ([10, 10], [-2, 1], [(slice(10, 20), 1, 1.0)]),
            ([2 ** 31 - 1] * 4, [0] * 4, [(slice(0, 40), 0, 1.0)])):
        plan.plan(lengths, adapters, None, m)
        y = ctx.linear_requests(w, x, bank, plan)
        with pytest.raises(MPError, match="out of range") as e:
            ctx.sync_check()
        assert e.value.status == 1
        ry, by, _, _ = _forward_ref(x, w64, wround, fac, segs, bank.rank_pad)
        _within("y", y, ry, by)
    ctx.sync_check()
    for h in (w, bank, plan):
        h.free()


def _grad_ref(x, dy, w, wround, fac, segs, v, cap, max_rank):
    m, k = x.shape
    n = dy.shape[1]
    x, dy, v = x.double(), dy.double(), v.double()
    wt = w.T
    dx = dy @ w
    mag = dy.abs() @ w.abs()
    err = wround * mag
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=x.device)  # noqa: E731
    da, db, ea, eb = z(cap, max_rank, k), z(cap, n, max_rank), z(cap, max_rank, k), z(cap, n, max_rank)
    for rows, a, s in segs:
        fa, fb = fac[a]
        r = fa.shape[0]
        u = s * (dy[rows] @ fb)
        ue = (n + 2) * ADD * abs(s) * (dy[rows].abs() @ fb.abs())
        dx[rows] += u @ fa
        low = u.abs() @ fa.abs()
        err[rows] += BF * low + ue @ fa.abs()
        mag[rows] += low
        da[a, :r] += u.T @ x[rows]
        ea[a, :r] += ((2.0 ** -16 + m * ADD) * u.abs() + ue).T @ x[rows].abs()
        db[a] += dy[rows].T @ v[rows, :max_rank]
        eb[a] += (2.0 ** -16 + m * ADD) * (dy[rows].abs().T @ v[rows, :max_rank].abs())
    err += (n + 128) * ADD * mag
    return (dx, err * (1 + 4 * BF) + BF * dx.abs() + 1e-30), (da, ea + 1e-30), (db, eb + 1e-30)


@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("saved", [16, 8])
@pytest.mark.parametrize("case", CASES, ids=[f"m{c[0]}_n{c[1]}_k{c[2]}_r{c[4]}" for c in CASES])
def test_linear_requests_grad(ctx, bits, saved, case):
    m, n, k, cap, max_rank, lengths, adapters, strengths = case
    rng = np.random.default_rng(2 * m + n + bits)
    w, w64, wround = _weight(ctx, rng, n, k, bits)
    ranks = [max(1, max_rank >> (i % 3)) for i in range(cap)]
    bank, fac = _bank(ctx, rng, n, k, cap, max_rank, ranks, training=True)
    plan = ctx.requests(len(lengths), m, cap)
    plan.plan(lengths, adapters, strengths, m)
    x, dy = _bf16(rng, m, k), _bf16(rng, m, n, scale=0.1)
    wt = ctx.transposed(w)
    _, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
    kept, x_in = x, x
    if saved == 8:
        x_in = ctx.checkpoint(x)
        kept = x_in.codes.double() * x_in.scales.double().repeat_interleave(128, 1)[:, :k]
    dx, da, db = ctx.linear_requests_grad(wt, dy, x_in, v, bank, plan)
    ctx.sync_check()
    segs = list(_segments(m, lengths, adapters, strengths))
    rx, ra, rb = _grad_ref(kept, dy, w64, wround, fac, segs, v, cap, max_rank)
    _within("dx", dx, *rx)
    _within("da", da, *ra)
    _within("db", db, *rb)
    for a in set(range(cap)) - {a for _, a, _ in segs}:
        assert not da[a].any() and not db[a].any(), "an adapter without rows has zero gradients"
    only_dx, none_a, none_b = ctx.linear_requests_grad(wt, dy, None, None, bank, plan, need_factors=False)
    none_x, only_da, only_db = ctx.linear_requests_grad(wt, dy, x_in, v[:, :max_rank], bank, plan, need_dx=False)
    assert none_a is None and none_b is None and none_x is None
    assert torch.equal(only_dx, dx) and torch.equal(only_da, da) and torch.equal(only_db, db)
    for h in (w, wt, bank, plan):
        h.free()


def test_transposed_weight_is_the_forward_weight(ctx):
    """The transpose holds the values the projections multiply with: unit rows
    through the transposed weight give the weight's columns as the forward has them."""
    rng = np.random.default_rng(8)
    for bits, mode in ((0, 0), (8, 0), (4, 0), (8, MP_QUANT_SYMMETRIC)):
        n, k = 192, 128
        w, w64, wround = _weight(ctx, rng, n, k, bits, mode)
        wt = ctx.transposed(w)
        eye_k = torch.eye(k, dtype=torch.bfloat16, device="cuda")
        eye_n = torch.eye(n, dtype=torch.bfloat16, device="cuda")
        fwd, bwd = ctx.linear(w, eye_k), ctx.linear(wt, eye_n)
        ctx.sync_check()
        assert torch.equal(fwd.T, bwd)
        assert ((bwd.double() - w64).abs() <= BF * w64.abs() * (1 + BF) + 1e-6 * w64.abs().max()).all()
        w.free()
        wt.free()


def test_gradient_against_differences(ctx):
    """The loss <y, g> is linear in A (B fixed) and in B (A fixed), so a change d
    of a factor moves it by <gradient, d>, up to the forward's own bound."""
    rng = np.random.default_rng(12)
    m, n, k, r = 200, 256, 192, 16
    w, w64, wround = _weight(ctx, rng, n, k, 0)
    bank, fac = _bank(ctx, rng, n, k, 2, r, [r, r], training=True)
    plan = ctx.requests(3, m, 2)
    lengths, adapters, strengths = [90, 40, 70], [0, 1, 0], [1.0, 0.5, -0.6]
    plan.plan(lengths, adapters, strengths, m)
    segs = list(_segments(m, lengths, adapters, strengths))
    x, g = _bf16(rng, m, k), _bf16(rng, m, n)
    y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
    wt = ctx.transposed(w)
    dx, da, db = ctx.linear_requests_grad(wt, g, x, v, bank, plan)
    loss = (y.double() * g.double()).sum()
    _, by0, _, _ = _forward_ref(x, w64, wround, fac, segs, bank.rank_pad)
    a, b = fac[0]
    for which, grad in (("a", da[0]), ("b", db[0])):
        old = a if which == "a" else b
        step = (grad.double() * (4.0 * old.std() / grad.double().std())).to(torch.bfloat16).double()
        a2, b2 = (a + step, b) if which == "a" else (a, b + step)
        a2, b2 = a2.to(torch.bfloat16), b2.to(torch.bfloat16)
        bank.set(0, a2, b2)
        y2 = ctx.linear_requests(w, x, bank, plan)
        _, by2, _, _ = _forward_ref(x, w64, wround, [(a2.double(), b2.double()), fac[1]], segs, bank.rank_pad)
        moved = (y2.double() * g.double()).sum() - loss
        taken = (a2.double() - a) if which == "a" else (b2.double() - b)
        foretold = (grad.double() * taken).sum()
        # the bounds of the outputs add up like the roundings they bound: at
        # random, so six times the root of the sum of squares is allowed
        slack = 6.0 * (((by0 + by2) * g.double().abs()) ** 2).sum().sqrt()
        assert foretold > 20 * slack, "the step has to stand out of the roundings"
        assert (moved - foretold).abs() <= slack
        bank.set(0, a.to(torch.bfloat16), b.to(torch.bfloat16))
    # dx: the loss is linear in x too
    step = (dx.double() * (0.5 * x.double().std() / dx.double().std()))
    x2 = (x.double() + step).to(torch.bfloat16)
    y2 = ctx.linear_requests(w, x2, bank, plan)
    _, by2, _, _ = _forward_ref(x2, w64, wround, fac, segs, bank.rank_pad)
    slack = 6.0 * ((((by0 + by2) * g.double().abs()) ** 2).sum().sqrt()
                   + ((BF * 4 * dx.double().abs() * (x2.double() - x.double()).abs()) ** 2).sum().sqrt())
    moved = (y2.double() * g.double()).sum() - loss
    foretold = (dx.double() * (x2.double() - x.double())).sum()
    assert foretold > 20 * slack and (moved - foretold).abs() <= slack
    ctx.sync_check()
    for h in (w, wt, bank, plan):
        h.free()


def test_offsets_past_32_bits(ctx):
    """The last adapter of a bank whose factors take more than 2^31 elements."""
    rng = np.random.default_rng(4)
    m, n, k, cap, r = 9, 128, 8704, 2048, 128
    assert cap * r * k > 2 ** 31
    w, w64, wround = _weight(ctx, rng, n, k, 0)
    bank = ctx.adapters(n, k, cap, r)
    a, b = _bf16(rng, r, k, scale=1 / math.sqrt(k)), _bf16(rng, n, r, scale=0.05)
    bank.set(cap - 1, a, b)
    plan = ctx.requests(2, m, cap)
    for mm, lengths in ((m, [4, 5]),):
        plan.plan(lengths, [cap - 1, cap - 2], None, mm)
        x = _bf16(rng, mm, k)
        y = ctx.linear_requests(w, x, bank, plan)
        ctx.sync_check()
        ry, by, _, _ = _forward_ref(x, w64, wround, {cap - 1: (a.double(), b.double())},
                                    [(slice(0, lengths[0]), cap - 1, 1.0)], bank.rank_pad)
        _within("y", y, ry, by)
    for h in (w, bank, plan):
        h.free()


@pytest.mark.parametrize("m", [6, 260])
def test_streams_and_graphs(ctx, m):
    """A call on another stream; and a graph captured once, replayed after the
    batch was planned again and an adapter replaced."""
    rng = np.random.default_rng(m)
    n, k, cap, r = 256, 128, 3, 16
    w, _, _ = _weight(ctx, rng, n, k, 8)
    bank, fac = _bank(ctx, rng, n, k, cap, r, [r] * cap, training=True)
    plan = ctx.requests(3, m, cap)
    third = m // 3
    len_d = torch.tensor([third, third, third], dtype=torch.int32, device="cuda")
    ad_d = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    s_d = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    x, dy = _bf16(rng, m, k), _bf16(rng, m, n)
    wt = ctx.transposed(w)

    def step():
        plan.plan(len_d, ad_d, s_d, m)
        y, v = ctx.linear_requests(w, x, bank, plan, ranks=True)
        saved = ctx.checkpoint(x)
        return (y, ctx.restore(saved)) + ctx.linear_requests_grad(wt, dy, saved, v, bank, plan)

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    len_d.copy_(torch.tensor([m - 2, 1, 1], dtype=torch.int32))
    ad_d.copy_(torch.tensor([2, -1, 0], dtype=torch.int32))
    x.copy_(_bf16(rng, m, k))
    bank.set(2, fac[0][0].to(torch.bfloat16), fac[1][1].to(torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    kept = [t.clone() for t in outs]
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, kept))
    ctx.sync_check()
    for h in (w, wt, bank, plan):
        h.free()


# ---- checkpoints -----------------------------------------------------------------

def _codes_ref(x32):
    """Codes and scales of f32 rows by the definition, in numpy f32."""
    m, k = x32.shape
    g = (k + 127) // 128
    pad = np.zeros((m, g * 128), np.float32)
    pad[:, :k] = x32
    x3 = pad.reshape(m, g, 128)
    with np.errstate(all="ignore"):
        top = np.abs(x3).max(-1)
        fin = np.isfinite(x3).all(-1)
        live = fin & (top >= np.float32(2.0 ** -110))
        inv = np.where(live, np.float32(127) * (np.float32(1) / top), np.float32(0)).astype(np.float32)
        q = np.where(live[..., None], np.rint(np.where(live[..., None], x3, 0) * inv[..., None]), 0)
        scale = np.where(fin, np.where(live, top / np.float32(127), np.float32(0)), np.float32(np.nan))
    return q.reshape(m, -1)[:, :k].astype(np.int8), scale.astype(np.float32)


@pytest.mark.parametrize("m,k,ld", [(1, 1, 8), (1, 128, 128), (3, 127, 128), (5, 129, 136), (17, 1000, 1000),
                                    (64, 3840, 3840), (2, 10240, 10256), (700, 200, 256)])
def test_checkpoint_codes(ctx, m, k, ld):
    rng = np.random.default_rng(m * 7 + k)
    big = rng.normal(size=(m, ld)).astype(np.float32) * np.exp(rng.uniform(-20, 20, size=(m, 1))).astype(np.float32)
    x = torch.from_numpy(big).to(torch.bfloat16).cuda()[:, :k]
    saved = ctx.checkpoint(x)
    back = ctx.restore(saved)
    ctx.sync_check()
    q, scale = _codes_ref(x.float().cpu().numpy())
    assert np.array_equal(saved.codes.cpu().numpy(), q)
    assert np.array_equal(saved.scales.cpu().numpy(), scale)
    want = torch.from_numpy(q.astype(np.float32) * np.repeat(scale, 128, 1)[:, :k]).to(torch.bfloat16)
    assert torch.equal(back.cpu(), want)
    # half a step of the group's scale, and the rounding to bf16
    step = torch.from_numpy(np.repeat(scale, 128, 1)[:, :k])
    assert ((back.cpu().double() - x.cpu().double()).abs() <= 0.5 * step * (1 + 1e-6) + BF * back.cpu().abs()).all()


def test_checkpoint_special_values(ctx):
    x = torch.zeros(8, 256, dtype=torch.bfloat16, device="cuda")
    x[0, 0] = float("inf")
    x[1, 130] = float("nan")
    x[2, :] = -3.3895e38
    x[3, 5] = 2.0 ** -111
    x[4, 5] = 2.0 ** -110
    x[5, 7], x[5, 8] = -0.0, 1.0
    x[6, :] = torch.arange(256, device="cuda").to(torch.bfloat16) - 127.5  # ties between codes
    saved = ctx.checkpoint(x)
    back = ctx.restore(saved).cpu()
    ctx.sync_check()
    q, scale = _codes_ref(x.float().cpu().numpy())
    assert np.array_equal(saved.codes.cpu().numpy(), q)
    assert np.array_equal(saved.scales.cpu().numpy(), scale, equal_nan=True)
    assert torch.isnan(back[0, :128]).all() and not back[0, 128:].any()
    assert not back[1, :128].any() and torch.isnan(back[1, 128:]).all()
    assert torch.equal(back[2], x[2].cpu()) and not back[3].any() and back[4, 5] == 2.0 ** -110


# ---- refusals --------------------------------------------------------------------

def test_refusals(ctx):
    rng = np.random.default_rng(1)
    n, k, m = 128, 64, 10
    for bad in (dict(capacity=0), dict(max_rank=0), dict(max_rank=129), dict(n=0), dict(capacity=5000)):
        args = dict(n=n, k=k, capacity=2, max_rank=8) | bad
        with pytest.raises(MPError):
            ctx.adapters(**args)
    for bad in ((0, 10, 2), (5000, 10, 2), (3, 0, 2), (3, 2 ** 19, 2), (3, 10, 0)):
        with pytest.raises(MPError):
            ctx.requests(*bad)
    w, _, _ = _weight(ctx, rng, n, k, 8)
    bank, _ = _bank(ctx, rng, n, k, 2, 8, [8, 4])
    train, _ = _bank(ctx, rng, n, k, 2, 8, [8, 4], training=True)
    plan = ctx.requests(2, m, 2)
    x, dy = _bf16(rng, m, k), _bf16(rng, m, n)
    a, b = _bf16(rng, 8, k), _bf16(rng, n, 8)
    with pytest.raises(MPError, match="outside"):
        bank.set(2, a, b)
    with pytest.raises(MPError, match="do not fit"):
        bank.set(0, a, b[:64])
    with pytest.raises(MPError, match="rank"):
        bank.set(0, _bf16(rng, 9, k), _bf16(rng, n, 9))
    with pytest.raises(MPError, match="not been planned"):
        ctx.linear_requests(w, x, bank, plan)
    with pytest.raises(MPError):
        plan.plan([1, 1, 1], [0, 0, 0], None, m)
    with pytest.raises(MPError):
        plan.plan([1, 1], [0, 0], None, m + 1)
    with pytest.raises(ValueError):
        plan.plan([1, 1], [0], None, m)
    plan.plan([5, 5], [0, 1], None, m)
    with pytest.raises(MPError, match="planned"):
        ctx.linear_requests(w, x[:9], bank, plan)
    with pytest.raises(ValueError):
        ctx.linear_requests(w, x.float(), bank, plan)
    with pytest.raises(ValueError):
        ctx.linear_requests(w, x[:, :32], bank, plan)
    with pytest.raises(ValueError):
        ctx.linear_requests(w, x.cpu(), bank, plan)
    with pytest.raises(ValueError):
        ctx.linear_requests(w, x, bank, plan, ranks=torch.empty(m, 8, device="cuda"))
    shifted = torch.empty(m * k + 1, dtype=torch.bfloat16, device="cuda")[1:].view(m, k)
    with pytest.raises(MPError, match="aligned"):
        ctx.linear_requests(w, shifted, bank, plan)
    other, _ = _bank(ctx, rng, n, 128, 2, 8, [8])
    with pytest.raises(MPError, match="adapters are for"):
        ctx.linear_requests(w, x, other, plan)
    small, _ = _bank(ctx, rng, n, k, 1, 8, [8])
    with pytest.raises(MPError, match="plan allows"):
        ctx.linear_requests(w, x, small, plan)
    _, v = ctx.linear_requests(w, x, train, plan, ranks=True)
    wt = ctx.transposed(w)
    with pytest.raises(MPError, match="training"):
        ctx.linear_requests_grad(wt, dy, x, v, bank, plan)
    with pytest.raises(MPError, match="dense"):
        sq, _, _ = _weight(ctx, rng, k, n, 8)
        ctx.linear_requests_grad(sq, dy, x, v, train, plan)
    with pytest.raises(ValueError):
        ctx.linear_requests_grad(wt, dy, x, v[:, :4], train, plan)
    with pytest.raises(ValueError):
        ctx.linear_requests_grad(wt, dy, x[:, :32], v, train, plan)
    saved = ctx.checkpoint(x)
    with pytest.raises(ValueError):
        ctx.linear_requests_grad(wt, dy, Checkpoint(saved.codes, saved.scales.contiguous().clone()[:5]), v, train, plan)
    with pytest.raises(ValueError):
        ctx.checkpoint(x.float())
    ctx.sync_check()
    for h in (w, wt, sq, bank, train, other, small, plan):
        h.free()
