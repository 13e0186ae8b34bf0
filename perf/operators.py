"""Cases for the operators that serve and train many low-rank adapters beside one shared projection.

Three operators, each in its plain form (elementary torch operations in 32 bits, rounded once at the end) and as the
calls a user makes of the framework:

  apply       y = x W^T + s_q (x A_q^T) B_q^T for the rows of every request q, W a packed or dense projection weight;
              with "train" also the rank-space rows v = s_q x A_q^T that the backward pass reads
  grad        from dy, v and x (or its 8-bit checkpoint): dx = dy W + s_q (dy B_q) A_q and, summed over the requests of
              each adapter, dA = (s_q dy B_q)^T x and dB = dy^T v
  checkpoint  x in 8 bits (a scale for every 128 features of a row) and back to bf16

The rows of a batch belong to requests of ragged lengths, one after the other; a request names its adapter (-1: none)
and its strength; rows after the last request have no adapter.
"""
import math
import sys
from pathlib import Path

import torch

own = False

GROUP = 64    # features that share a scale and a bias in a packed weight
CK_GROUP = 128  # features that share a scale in an 8-bit checkpoint
CK_TINY = 2.0 ** -110  # groups below this are stored as zeros


# ---- cases -----------------------------------------------------------------------------------------------------

def listed():
    a = dict(kind="apply", train=False, pad=0)
    g = dict(kind="grad", pad=0)
    return [
        # one new token of one request
        dict(a, name="apply_1_token", m=1, n=3840, k=3840, bits=8, requests=1, cap=8, rank=16, mix=1),
        # a step of single tokens, each request with an adapter of its own
        dict(a, name="apply_16_tokens", m=16, n=10240, k=3840, bits=4, requests=16, cap=16, rank=32, mix=2),
        # short ragged prompts; some requests without an adapter, one empty
        dict(a, name="apply_short_prompts", m=517, n=3840, k=10240, bits=8, requests=13, cap=8, rank=64, mix=3),
        # small dense layer in training, odd sizes, rows of x and y not packed
        dict(a, name="apply_train_odd", train=True, pad=3, m=333, n=648, k=640, bits=0, requests=5, cap=4, rank=24, mix=4),
        # a batch of images' tokens, one request each
        dict(a, name="apply_4352_rows", m=4352, n=3840, k=3840, bits=8, requests=8, cap=8, rank=32, mix=5),
        # the largest projection over the longest batch
        dict(a, name="apply_16896_rows", m=16896, n=10240, k=3840, bits=4, requests=8, cap=8, rank=32, mix=6),
        # backward pass of a small layer, odd sizes
        dict(g, name="grad_small", m=77, n=384, k=640, bits=0, requests=3, cap=4, rank=8, saved=16, pad=1, mix=7),
        # backward pass of an attention projection over four images' rows, x from its 8-bit checkpoint
        dict(g, name="grad_4352_saved8", m=4352, n=3840, k=3840, bits=8, requests=4, cap=4, rank=16, saved=8, mix=8),
        # the same over a long batch of many requests, x kept in bf16
        dict(g, name="grad_16896_rows", m=16896, n=3840, k=3840, bits=0, requests=24, cap=16, rank=64, saved=16, mix=9),
        # activations of a caption, of an attention input and of the widest layer's input
        dict(kind="checkpoint", name="checkpoint_256", m=256, k=3840, pad=0),
        dict(kind="checkpoint", name="checkpoint_odd", m=1001, k=10216, pad=2),
        dict(kind="checkpoint", name="checkpoint_16896", m=16896, k=10240, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(n):
    """Layer widths come from the shapes of this library's own layers and what lies between them."""
    return n + GROUP if n == 3072 else n


def draw(rng):
    kind = rng.choice(["apply", "apply", "apply", "grad", "grad", "checkpoint"])
    m = _log(rng, 1, 16896)
    if kind == "checkpoint":
        return dict(kind=kind, m=m, k=_width(8 * _log(rng, 8, 1280)), pad=rng.choice([0, 0, 1, 5]))
    n, k = _width(8 * _log(rng, 16, 1280)), _width(GROUP * _log(rng, 2, 160))
    m = min(m, 16896 * 10240 * 3840 // (n * k))  # no more than the largest listed product
    c = dict(kind=kind, m=m, n=n, k=k, bits=rng.choice([0, 4, 8]), requests=min(m + 1, _log(rng, 1, 48)),
             cap=_log(rng, 1, 16), rank=4 * rng.randint(1, 16), mix=rng.randrange(1 << 20), pad=rng.choice([0, 0, 1, 4]))
    if kind == "apply":
        return dict(c, train=rng.random() < 0.3)
    return dict(c, saved=rng.choice([8, 16]))


def layout(c):
    """(lengths, adapters, strengths, ranks) of a case: plain lists, from the case alone."""
    import random
    r = random.Random(c["mix"])
    m, q = c["m"], c["requests"]
    if q >= m:
        lengths = [1] * m + [0] * (q - m)
    else:
        empty = 2 if q > 4 else -1  # a request that has nothing in this batch
        w = [0.0 if i == empty else r.uniform(0.3, 1.7) for i in range(q)]
        whole = m if q == 1 else m - m // 50  # rows past the last request have no adapter
        lengths = [int(whole * v / sum(w)) for v in w]
    adapters = [r.randrange(c["cap"]) if i % 7 != 3 else -1 for i in range(q)]
    strengths = [round(r.uniform(-0.5, 1.5), 3) if i % 11 != 5 else 0.0 for i in range(q)]
    ranks = [max(1, c["rank"] >> (i % 3)) for i in range(c["cap"])]
    return lengths, adapters, strengths, ranks


# ---- inputs ----------------------------------------------------------------------------------------------------

def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


def _rows(g, m, k, pad, dev, scale=1.0):
    """bf16 activations [m, k], a few features much larger than the rest; row pitch k + 8 pad rounded up to 8."""
    ld = (k + 7) // 8 * 8 + 8 * pad
    wide = 1.0 + 9.0 * (torch.rand(ld, generator=g, device=dev) < 0.01)
    x = torch.randn(m, ld, generator=g, device=dev) * wide * scale
    return x.to(torch.bfloat16)[:, :k]


def _inputs(c, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(int(seed))
    m, k, pad = c["m"], c["k"], c["pad"]
    d = {"case": c, "dev": dev}
    if c["kind"] == "checkpoint":
        return dict(d, x=_rows(g, m, k, pad, dev))
    n, bits, cap, rank = c["n"], c["bits"], c["cap"], c["rank"]
    lengths, adapters, strengths, ranks = layout(c)
    std = 1.0 / math.sqrt(k)
    if bits:
        top = 2 ** bits - 1
        d["codes"] = torch.randint(0, top + 1, (n, k), generator=g, device=dev, dtype=torch.int32)
        step = std * (12.0 ** 0.5) / top * (0.75 + 0.5 * torch.rand(n, k // GROUP, generator=g, device=dev))
        d["scales"] = step.to(torch.bfloat16)
        d["biases"] = (-step * top / 2 + 0.1 * std * torch.randn(n, k // GROUP, generator=g, device=dev)).to(torch.bfloat16)
    else:
        d["weight"] = (torch.randn(n, k, generator=g, device=dev) * std).to(torch.bfloat16)
    d["a"] = [(torch.randn(r, k, generator=g, device=dev) * std).to(torch.bfloat16) for r in ranks]
    d["b"] = [(torch.randn(n, r, generator=g, device=dev) * 0.5 / math.sqrt(r)).to(torch.bfloat16) for r in ranks]
    d["x"] = _rows(g, m, k, pad, dev)
    d["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
    d["adapters"] = torch.tensor(adapters, dtype=torch.int32, device=dev)
    d["strengths"] = torch.tensor(strengths, dtype=torch.float32, device=dev)
    if c["kind"] == "grad":
        d["dy"] = _rows(g, m, n, pad, dev, 0.05)
        # the rank-space rows the forward pass kept: zero where a row has no adapter
        v = torch.randn(m, rank, generator=g, device=dev)
        row, s = _row_adapter(d)
        width = torch.tensor(ranks + [0], device=dev)[row]  # the last entry: no adapter
        d["v"] = v * s[:, None] * (torch.arange(rank, device=dev)[None] < width[:, None])
        if c["saved"] == 8:
            d["q"], d["q_scale"] = _to_8_bits(d["x"])
    return d


def _row_adapter(d):
    """Adapter (-1: none) and strength (0 there) of every row of the batch."""
    m = d["case"]["m"]
    lengths = d["lengths"].long()
    left = max(0, m - int(sum(layout(d["case"])[0])))
    pad_a = torch.full((left,), -1, dtype=torch.int32, device=d["dev"])
    row = torch.cat([torch.repeat_interleave(d["adapters"], lengths, output_size=m - left), pad_a]).long()
    s = torch.cat([torch.repeat_interleave(d["strengths"], lengths, output_size=m - left),
                   torch.zeros(left, device=d["dev"])])
    return row, torch.where(row >= 0, s, torch.zeros_like(s))


def _groups(x):
    """[m, k] as [m, groups, CK_GROUP], zeros after a ragged end."""
    m, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % CK_GROUP))
    return x.reshape(m, -1, CK_GROUP)


def _to_8_bits(x):
    """Codes [m, k] and scales [m, groups]: scale = max|x| / 127, code = the nearest whole number to x (127 / max|x|)."""
    x3 = _groups(x)
    top = x3.abs().amax(-1)
    live = top >= CK_TINY
    scale = torch.where(live, top / 127.0, torch.zeros_like(top))
    inv = torch.where(live, 127.0 / top, torch.zeros_like(top))
    q = torch.round(x3 * inv[..., None]).to(torch.int8)
    return q.reshape(x.shape[0], -1)[:, :x.shape[1]], scale


def _from_8_bits(q, scale):
    k = q.shape[1]
    return (_groups(q) * scale[..., None]).reshape(q.shape[0], -1)[:, :k]


# ---- the framework's side --------------------------------------------------------------------------------------

_ctx = None


class _Handles:
    """The library handles a program keeps, freed with the state that holds them."""

    def __init__(self, *handles):
        self.handles = handles

    def __del__(self):
        for h in self.handles:
            h.free()


def _context():
    global _ctx
    if _ctx is None:
        package = str(Path.cwd() / "vpipe-ming-image_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from mingproj.proj import Context
        _ctx = Context(torch.cuda.current_device())
    return _ctx


def _pack(codes, bits):
    """Codes [n, k] as the 32-bit words of a packed weight, first code in the low bits."""
    per = 32 // bits
    w = codes.reshape(codes.shape[0], -1, per).long()
    return (w << (bits * torch.arange(per, device=codes.device))).sum(-1).to(torch.int32)


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "checkpoint":
        if own:
            _context()
        return d
    n, k, cap, rank = case["n"], case["k"], case["cap"], case["rank"]
    if own:  # the weight, the adapters and the batch's plan, as a program keeps them
        ctx = _context()
        if case["bits"]:
            w = ctx.upload(n, k, case["bits"], _pack(d["codes"], case["bits"]), d["scales"], d["biases"])
        else:
            w = ctx.upload(n, k, 0, d["weight"])
        train = case["kind"] == "grad"
        bank = ctx.adapters(n, k, cap, rank, training=train)
        for i, (a, b) in enumerate(zip(d["a"], d["b"])):
            bank.set(i, a, b)
        plan = ctx.requests(case["requests"], case["m"], cap)
        plan.plan(d["lengths"], d["adapters"], d["strengths"], case["m"])
        d.update(w=w, bank=bank, plan=plan)
        kept = [w, bank, plan]
        if train:
            d["wt"] = ctx.transposed(w)
            kept.append(d["wt"])
            if case["saved"] == 8:
                d["saved"] = ctx.checkpoint(d["x"])
        d["kept"] = _Handles(*kept)
    else:  # dense 32-bit matrices: the weight, and all adapters' factors as one
        if case["bits"]:
            w = d["codes"].float().reshape(n, -1, GROUP) * d["scales"].float()[..., None] + d["biases"].float()[..., None]
            d["w32"] = w.reshape(n, k)
        else:
            d["w32"] = d["weight"].float()
        a = torch.zeros(cap, rank, k, device=d["dev"])
        b = torch.zeros(n, cap, rank, device=d["dev"])
        for i, (fa, fb) in enumerate(zip(d["a"], d["b"])):
            a[i, :fa.shape[0]] = fa
            b[:, i, :fb.shape[1]] = fb
        d["a32"], d["b32"] = a.reshape(cap * rank, k), b.reshape(n, cap * rank)
    d.pop("codes", None)
    return d


# ---- one pass --------------------------------------------------------------------------------------------------

def run(d):
    return (_run_own if own else _run_plain)(d)


def _run_own(d):
    c, ctx = d["case"], _context()
    if c["kind"] == "checkpoint":
        saved = ctx.checkpoint(d["x"])
        return {"x": ctx.restore(saved), "scale": saved.scales}
    if c["kind"] == "apply":
        if c["train"]:
            y, v = ctx.linear_requests(d["w"], d["x"], d["bank"], d["plan"], ranks=True)
            return {"y": y, "v": v[:, :c["rank"]]}
        return {"y": ctx.linear_requests(d["w"], d["x"], d["bank"], d["plan"])}
    x = d["saved"] if c["saved"] == 8 else d["x"]
    dx, da, db = ctx.linear_requests_grad(d["wt"], d["dy"], x, d["v"], d["bank"], d["plan"])
    return {"dx": dx, "da": da, "db": db}


def _run_plain(d):
    c = d["case"]
    if c["kind"] == "checkpoint":
        q, scale = _to_8_bits(d["x"])
        return {"x": _from_8_bits(q, scale).to(torch.bfloat16), "scale": scale}
    m, n, k, cap, rank = c["m"], c["n"], c["k"], c["cap"], c["rank"]
    row, s = _row_adapter(d)
    # every adapter's rank-space columns for every row, then only the row's own
    mine = (row[:, None] == torch.arange(cap, device=d["dev"])[None]).float()
    if c["kind"] == "apply":
        x = d["x"].float()
        v = (x @ d["a32"].T).reshape(m, cap, rank) * (mine * s[:, None])[..., None]
        y = (x @ d["w32"].T + v.reshape(m, cap * rank) @ d["b32"].T).to(torch.bfloat16)
        return {"y": y, "v": v.sum(1)} if c["train"] else {"y": y}
    dy = d["dy"].float()
    x = _from_8_bits(d["q"], d["q_scale"]) if c["saved"] == 8 else d["x"].float()
    u = ((dy @ d["b32"]).reshape(m, cap, rank) * (mine * s[:, None])[..., None]).reshape(m, cap * rank)
    v = (d["v"][:, None] * mine[..., None]).reshape(m, cap * rank)
    return {"dx": (dy @ d["w32"] + u @ d["a32"]).to(torch.bfloat16),
            "da": (u.T @ x).reshape(cap, rank, k),
            "db": (dy.T @ v).reshape(n, cap, rank).permute(1, 0, 2).contiguous()}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    d = _inputs(case, seed)
    x = d["x"].double()
    if case["kind"] == "checkpoint":
        back, scales = [], []
        for lo in range(0, case["k"], CK_GROUP):  # the codes are chosen in 32 bits, by definition
            part = d["x"][:, lo:lo + CK_GROUP].float()
            top = part.abs().max(dim=1, keepdim=True).values
            live = top >= CK_TINY
            code = torch.round(part * torch.where(live, 127.0 / top, top * 0)).double()
            scale = torch.where(live, top.double() / 127.0, top.double() * 0)
            back.append(code * scale)
            scales.append(scale)
        return {"x": torch.cat(back, 1), "scale": torch.cat(scales, 1)}
    lengths, adapters, strengths, ranks = layout(case)
    if case["bits"]:
        w = d["codes"].double()
        w *= d["scales"].double().repeat_interleave(GROUP, 1)
        w += d["biases"].double().repeat_interleave(GROUP, 1)
    else:
        w = d["weight"].double()
    if case["kind"] == "apply":
        y = x @ w.T
        v = torch.zeros(case["m"], case["rank"], dtype=torch.float64, device=d["dev"])
        at = 0
        for length, i, s in zip(lengths, adapters, strengths):
            rows = slice(at, at + length)
            at += length
            if i >= 0 and length:
                t = s * (x[rows] @ d["a"][i].double().T)
                y[rows] += t @ d["b"][i].double().T
                v[rows, :ranks[i]] = t
        return {"y": y, "v": v} if case["train"] else {"y": y}
    if case["saved"] == 8:
        q, scale = d["q"].double(), d["q_scale"].double()
        x = q * scale.repeat_interleave(CK_GROUP, 1)[:, :case["k"]]
    dy, v = d["dy"].double(), d["v"].double()
    dx = dy @ w
    da = torch.zeros(case["cap"], case["rank"], case["k"], dtype=torch.float64, device=d["dev"])
    db = torch.zeros(case["cap"], case["n"], case["rank"], dtype=torch.float64, device=d["dev"])
    at = 0
    for length, i, s in zip(lengths, adapters, strengths):
        rows = slice(at, at + length)
        at += length
        if i >= 0 and length:
            t = s * (dy[rows] @ d["b"][i].double())
            dx[rows] += t @ d["a"][i].double()
            da[i, :ranks[i]] += t.T @ x[rows]
            db[i, :, :ranks[i]] += dy[rows].T @ v[rows, :ranks[i]]
    return {"dx": dx, "da": da, "db": db}


def work(case):
    m, k = case["m"], case["k"]
    if case["kind"] == "checkpoint":
        # x once, the codes and scales that are kept, and the bf16 rows
        return {"bytes": m * k * (2 + 1 + 2) + 4 * m * -(-k // CK_GROUP), "flops": 0}
    n, bits = case["n"], case["bits"]
    lengths, adapters, strengths, ranks = layout(case)
    live = [(length, i) for length, i, s in zip(lengths, adapters, strengths) if i >= 0 and length and s]
    factors = 2 * (n + k) * sum(ranks[i] for i in {i for _, i in live})
    low = sum(2 * length * ranks[i] for length, i in live)
    if case["kind"] == "apply":
        weight = n * k * bits // 8 + 4 * n * (k // GROUP) if bits else 2 * n * k
        kept = 4 * m * case["rank"] if case["train"] else 0
        return {"bytes": weight + 2 * m * (n + k) + factors + kept, "flops": 2 * m * n * k + low * (n + k)}
    saved = 2 * m * k if case["saved"] == 16 else m * k + 4 * m * -(-k // CK_GROUP)
    grads = 4 * case["cap"] * case["rank"] * (n + k)
    return {"bytes": 2 * n * k + 2 * m * n + saved + 4 * m * case["rank"] + 2 * m * k + factors + grads,
            "flops": 2 * m * n * k + 2 * low * (n + k)}
