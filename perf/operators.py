"""The serving operators around the 8-bit paged K/V cache, as cases that can be timed.

Between the q/k/v projections and the output projection an engine places the new
tokens of its requests in cache pages ("slots"), rotates q and k ("rope"), writes
k and v into the pages ("append") and attends over them ("attn").  Each of these
is a case kind.  Where ``own`` is false a pass computes the operator with
elementary torch operations; where it is true, it calls gemmainfer_amd.ops.

Head shapes are those of the benchmark's decoder layers: a sliding-window layer
has 16 query heads and 8 kv heads of 256, a global layer 16 and 2 of 512; 64 and
128 are the generic head widths.  The cache holds e4m3 codes, K as
[pages, kv heads, page, D] and V as [pages, kv heads, D, page], with one fp32
scale (a power of two) per page and kv head.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# (query heads, kv heads, head width)
HEADS = {"sliding": (16, 8, 256), "global": (16, 2, 512), "wide": (32, 8, 128), "small": (12, 4, 64)}
F8_MAX = 448.0
MIN_EXP, MAX_EXP = -40, 40


def listed():
    return [
        # a decode step of a handful of requests: each places one token, latency alone
        {"name": "slots_decode", "kind": "slots", "B": 7, "ctx_lo": 100, "ctx_hi": 1500, "new_lo": 1, "new_hi": 1,
         "page": 16, "pad": 1},
        # a step that mixes prompts and decoded tokens of a few hundred requests
        {"name": "slots_mixed", "kind": "slots", "B": 301, "ctx_lo": 0, "ctx_hi": 4000, "new_lo": 0, "new_hi": 97,
         "page": 64, "pad": 37},
        # one decoded token far into a long context, a quarter of the head rotated
        {"name": "rope_decode", "kind": "rope", "T": 1, "heads": "global", "part": 0.25, "inter": False,
         "scaling": "yarn", "far": 900000, "dtype": "bf16"},
        # an ordinary prompt of a sliding-window layer
        {"name": "rope_prompt", "kind": "rope", "T": 2047, "heads": "sliding", "part": 1.0, "inter": False,
         "scaling": "none", "far": 0, "dtype": "bf16"},
        # a ragged prompt of an fp16 engine with interleaved pairs, frequencies stretched
        {"name": "rope_interleaved", "kind": "rope", "T": 777, "heads": "wide", "part": 0.5, "inter": True,
         "scaling": "linear", "far": 40000, "dtype": "fp16"},
        # a decode step of a batch: one row into each request's last page
        {"name": "append_decode", "kind": "append", "B": 61, "ctx_lo": 1, "ctx_hi": 700, "new_lo": 1, "new_hi": 1,
         "heads": "sliding", "page": 16, "dtype": "bf16"},
        # prompts of several requests, some onto pages that hold tokens
        {"name": "append_prompt", "kind": "append", "B": 5, "ctx_lo": 0, "ctx_hi": 300, "new_lo": 500, "new_hi": 1900,
         "heads": "sliding", "page": 64, "dtype": "bf16"},
        # one decoded token of one request behind a sliding window
        {"name": "attn_decode_one", "kind": "attn", "B": 1, "lo": 1391, "hi": 1391, "q": 1, "heads": "sliding",
         "page": 16, "window": 1024, "dtype": "bf16"},
        # a decode step of a ragged batch
        {"name": "attn_decode_batch", "kind": "attn", "B": 47, "lo": 33, "hi": 8190, "q": 1, "heads": "sliding",
         "page": 16, "window": 0, "dtype": "bf16"},
        # two very long contexts in a global layer: few rows, one long axis
        {"name": "attn_decode_long", "kind": "attn", "B": 2, "lo": 70001, "hi": 130005, "q": 1, "heads": "global",
         "page": 64, "window": 0, "dtype": "bf16"},
        # six draft tokens and one more of an fp16 engine, verified together
        {"name": "attn_verify", "kind": "attn", "B": 9, "lo": 600, "hi": 5000, "q": 7, "heads": "global",
         "page": 32, "window": 0, "dtype": "fp16"},
        # a chunk of a long prompt: the matrix cores' case
        {"name": "attn_prefill", "kind": "attn", "B": 1, "lo": 8100, "hi": 8100, "q": 2048, "heads": "sliding",
         "page": 64, "window": 0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["slots", "rope", "append", "append", "attn", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "slots":
        hi = _log(rng, 1, 100)
        return {"kind": kind, "B": _log(rng, 1, 600), "ctx_lo": 0, "ctx_hi": _log(rng, 10, 5000),
                "new_lo": rng.choice([0, 1]), "new_hi": hi, "page": page, "pad": rng.randint(0, 40)}
    heads = rng.choice(["sliding", "global", "wide", "small"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "rope":
        return {"kind": kind, "T": _log(rng, 1, 2047), "heads": heads, "part": rng.choice([0.25, 0.5, 1.0]),
                "inter": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "yarn"]),
                "far": _log(rng, 1, 1000000), "dtype": rng.choice([dtype, dtype, "fp32"])}
    if kind == "append":
        if rng.random() < 0.5:
            return {"kind": kind, "B": _log(rng, 1, 200), "ctx_lo": 0, "ctx_hi": _log(rng, 2, 600), "new_lo": 1,
                    "new_hi": rng.choice([1, 1, 7]), "heads": heads, "page": page,
                    "dtype": rng.choice([dtype, dtype, "fp32"])}
        hi = _log(rng, 20, 1900)
        return {"kind": kind, "B": rng.randint(1, 5), "ctx_lo": 0, "ctx_hi": _log(rng, 2, 300), "new_lo": hi // 3,
                "new_hi": hi, "heads": heads, "page": page, "dtype": dtype}
    window = rng.choice([0, 0, 0, 512, 1024])
    shape = rng.choice(["decode", "decode", "verify", "long", "prompt"])
    if shape == "decode":
        b, q, hi = _log(rng, 1, 60), 1, _log(rng, 10, 6000)
    elif shape == "verify":
        b, q, hi = _log(rng, 1, 12), rng.randint(2, 8), _log(rng, 20, 8000)
    elif shape == "long":
        b, q, hi = 1, rng.randint(1, 4), _log(rng, 10000, 100000)
    else:
        b, q = rng.randint(1, 3), _log(rng, 20, 800)
        hi = q + _log(rng, 1, 3000)
    return {"kind": kind, "B": b, "lo": max(q, hi // rng.randint(1, 9)), "hi": max(q, hi), "q": q, "heads": heads,
            "page": page, "window": window, "dtype": dtype}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 6151 + 29)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _spread(n, lo, hi):
    """n lengths over [lo, hi], in no order; the same for every seed."""
    step = next(s for s in (7919, 7907, 7901) if math.gcd(s, n) == 1)
    return [hi if n == 1 else lo + (hi - lo) * (i * step % n) // (n - 1) for i in range(n)]


def _lengths(case):
    b = case["B"]
    ctx = _spread(b, case["ctx_lo"], case["ctx_hi"])
    return ctx, _spread(b, case["new_lo"], case["new_hi"])[::-1]


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _pages(case, lens, g):
    """A block table (-1 behind each request's pages) over randomly placed pages, and the number of pages."""
    p = case["page"]
    need = [-(-n // p) for n in lens]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    cols = max(need) + 1
    col = torch.arange(cols, device=DEV)
    n = _int(need, torch.int64)
    first = torch.cumsum(n, 0) - n
    at = (first[:, None] + col[None]).clamp(max=total - 1)
    return torch.where(col[None] < n[:, None], perm[at], torch.full_like(at, -1, dtype=torch.int32)), total


def _powers(lo, hi):
    """2^lo ... 2^hi, each of them exact (exp2 and ldexp on the device need not be)."""
    return torch.tensor([2.0 ** e for e in range(lo, hi + 1)], device=DEV)


def _pow2_scale(amax):
    """The smallest power of two s with amax <= 448 s, at least 2^-40; NaN where no code can hold amax."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8).clamp(MIN_EXP, MAX_EXP)
    s = _powers(MIN_EXP, MAX_EXP)[torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).long() - MIN_EXP]
    bad = ~torch.isfinite(amax) | (amax > F8_MAX * 2.0 ** MAX_EXP)
    return torch.where(bad, torch.full_like(s, float("nan")), s)


def _cache(case, total, g):
    """Pages of random keys and values whose sizes differ by page and head."""
    _, hk, d = HEADS[case["heads"]]
    p = case["page"]
    k = _randn(g, total, hk, p, d) * torch.exp2(_randn(g, total, hk, 1, 1) * 0.5)
    v = _randn(g, total, hk, d, p) * torch.exp2(_randn(g, total, hk, 1, 1))
    r = {}
    for name, t in (("k", k), ("v", v)):
        s = _pow2_scale(t.abs().amax((2, 3)))
        r[name], r[name + "_scale"] = (t / s[:, :, None, None]).to(torch.float8_e4m3fn), s
    return r


def _frequencies(case):
    """Angle per position of each rotated pair (fp64), and the factor on cos and sin."""
    _, _, d = HEADS[case["heads"]]
    r = int(d * case["part"])
    i = torch.arange(0, r, 2, dtype=torch.float64, device=DEV)
    f, mscale = 1e4 ** (-i / r), 1.0
    if case["scaling"] == "linear":
        f = f / 8
    elif case["scaling"] == "yarn":
        factor, original = 16.0, 8192
        turns = original * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        f, mscale = f / factor * (1 - keep) + f * keep, 0.1 * math.log(factor) + 1
    return f, mscale


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["kind"] == "slots":
        ctx, new = _lengths(case)
        p = case["page"]
        table, total = _pages(case, ctx, g)
        need = sum(-(-(c + n) // p) - -(-c // p) for c, n in zip(ctx, new))
        cols = max(-(-(c + n) // p) for c, n in zip(ctx, new)) + 1
        wide = torch.full((case["B"], max(cols, table.shape[1])), -1, dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table
        free = total + torch.randperm(need + 9, generator=g, device=DEV).to(torch.int32)
        s.update(ctx=_int(ctx), new=_int(new), table=wide, free=free, used=_int([4, 0, 0]),
                 n=sum(new) + case["pad"])
        return s
    hq, hk, d = HEADS[case["heads"]]
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "rope":
        t = case["T"]
        f, mscale = _frequencies(case)
        s.update(q=_randn(g, t, hq, d).to(dt), k=_randn(g, t, hk, d).to(dt), freq=f, mscale=mscale,
                 pos=torch.arange(t, device=DEV) + case["far"])
        return s
    if case["kind"] == "append":
        ctx, new = _lengths(case)
        p = case["page"]
        table, total = _pages(case, [c + n for c, n in zip(ctx, new)], g)
        s.update(_cache(case, total, g))
        c, n = _int(ctx, torch.int64), _int(new, torch.int64)
        b = torch.repeat_interleave(torch.arange(case["B"], device=DEV), n)
        pos = torch.arange(b.numel(), device=DEV) - (torch.cumsum(n, 0) - n)[b] + c[b]
        s["slots"] = table[b, pos // p].long() * p + pos % p
        # rows of ordinary size, a few of them large: those raise the scales of pages that hold tokens
        size = torch.exp2(_randn(g, b.numel(), 1, 1) * 1.5)
        s["k_new"] = (_randn(g, b.numel(), hk, d) * size).to(dt)
        s["v_new"] = (_randn(g, b.numel(), hk, d) * size).to(dt)
        return s
    lens = _spread(case["B"], case["lo"], case["hi"])
    table, total = _pages(case, lens, g)
    s.update(_cache(case, total, g))
    s.update(table=table, lens=_int(lens), q=(1.5 * _randn(g, case["B"] * case["q"], hq, d)).to(dt),
             start=None if case["q"] == 1 else _int([i * case["q"] for i in range(case["B"] + 1)]),
             scale=d ** -0.5)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _own_cache(s):
    from gemmainfer_amd import ops
    return ops.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])


def _own_slots(s):
    from gemmainfer_amd import ops
    r = ops.kv_slots(s["ctx"], s["new"], s["table"], s["free"], s["used"], s["case"]["page"], s["n"])
    return {"slots": r.slots, "positions": r.positions, "q_start": r.q_start, "seq_lens": r.seq_lens,
            "status": r.status, "table": s["table"]}


def _own_rope(s):
    from gemmainfer_amd import ops
    q, k = ops.rope_rows(s["q"], s["k"], s["pos"], s["freq"], interleaved=s["case"]["inter"], mscale=s["mscale"])
    return {"q": q, "k": k}


def _own_append(s):
    from gemmainfer_amd import ops
    ops.kv_append(s["k_new"], s["v_new"], s["slots"], _own_cache(s))
    return {n: s[n] for n in ("k", "v", "k_scale", "v_scale")}


def _own_attn(s):
    from gemmainfer_amd import ops
    return ops.kv_attention(s["q"], _own_cache(s), s["table"], s["lens"], s["start"], scale=s["scale"],
                            window=s["case"]["window"])


_own = {"slots": _own_slots, "rope": _own_rope, "append": _own_append, "attn": _own_attn}


def _plain_slots(s):
    p, n, table = s["case"]["page"], s["n"], s["table"]
    cols = table.shape[1]
    ctx, new, used = s["ctx"].long().clamp(min=0), s["new"].long().clamp(min=0), s["used"][0].long()
    end = torch.cumsum(new, 0)
    start = (end - new).clamp(max=n)
    dropped = end[-1] - end[-1].clamp(max=n)
    new = torch.minimum(new, n - start)
    lens = ctx + new
    have, want = (ctx + p - 1) // p, (lens + p - 1) // p
    add = (want.clamp(max=cols) - have.clamp(max=cols))
    first = used + torch.cumsum(add, 0) - add
    col = torch.arange(cols, device=DEV)
    fresh = (col[None] >= have[:, None]) & (col[None] < want[:, None])
    at = first[:, None] + col[None] - have[:, None]
    page = torch.where(at < s["free"].numel(), s["free"][at.clamp(0, s["free"].numel() - 1)].long(), -1)
    table.copy_(torch.where(fresh, page, table.long()))
    q_start = torch.cat([start, (start + new)[-1:]])
    t = torch.arange(n, device=DEV)
    b = torch.searchsorted(q_start[1:], t, right=True).clamp(max=ctx.numel() - 1)
    live = t < q_start[-1]
    pos = torch.where(live, ctx[b] + t - start[b], 0)
    page = torch.where(pos // p < cols, table[b, (pos // p).clamp(max=cols - 1)].long(), -1)
    total = add.sum()
    got = torch.minimum(total, (s["free"].numel() - used).clamp(min=0))
    status = torch.stack([used + got, (want - have).sum() - got, dropped])
    return {"slots": torch.where(live & (page >= 0), page * p + pos % p, -1), "positions": pos,
            "q_start": q_start.int(), "seq_lens": lens.int(), "status": status.int(), "table": table}


def _plain_rope(s):
    case, f = s["case"], s["freq"]
    a = s["pos"].double()[:, None, None] * f
    cos, sin = (a.cos() * s["mscale"]).float(), (a.sin() * s["mscale"]).float()
    half = f.numel()

    def turn(x):
        y = x.float()
        if case["inter"]:
            u, w = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
            r = torch.stack([u * cos - w * sin, w * cos + u * sin], -1).flatten(-2)
        else:
            u, w = y[..., :half], y[..., half:2 * half]
            r = torch.cat([u * cos - w * sin, w * cos + u * sin], -1)
        return torch.cat([r, y[..., 2 * half:]], -1).to(x.dtype)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def _plain_append(s):
    p = s["case"]["page"]
    page, row = s["slots"] // p, s["slots"] % p
    pages = s["k"].shape[0]
    restart = torch.zeros(pages, dtype=torch.int64, device=DEV).index_add_(0, page, (row == 0).long()) > 0
    touched = torch.zeros(pages, dtype=torch.bool, device=DEV).index_fill_(0, page, True)
    for name, axis in (("k", 2), ("v", 3)):
        x, codes, old = s[name + "_new"].float(), s[name], s[name + "_scale"]
        amax = torch.zeros_like(old).index_reduce_(0, page, x.abs().amax(-1), "amax")
        need = _pow2_scale(amax)
        new = torch.where(restart[:, None], need, torch.maximum(old, need))
        new = torch.where(touched[:, None], new, old)
        grown = touched[:, None] & ~restart[:, None] & (new > old)
        ratio = torch.where(grown, old / new, torch.ones_like(old))
        moved = (codes.float() * ratio[:, :, None, None]).to(torch.float8_e4m3fn)
        rows = (x / new[page][..., None]).to(torch.float8_e4m3fn)
        moved = moved.view(torch.uint8)
        if axis == 2:
            moved[page, :, row, :] = rows.view(torch.uint8)
        else:
            moved[page, :, :, row] = rows.view(torch.uint8)
        codes.copy_(moved.view(torch.float8_e4m3fn))
        old.copy_(new)
    return {n: s[n] for n in ("k", "v", "k_scale", "v_scale")}


def _plain_attn(s):
    case, table = s["case"], s["table"]
    b, q, p = case["B"], case["q"], case["page"]
    hq, hk, d = HEADS[case["heads"]]
    cols = -(-case["hi"] // p)
    page = table[:, :cols].clamp(min=0).long()
    k = s["k"][page].float() * s["k_scale"][page][..., None, None]  # [B, cols, hk, p, d]
    v = s["v"][page].float() * s["v_scale"][page][..., None, None]  # [B, cols, hk, d, p]
    k = k.transpose(1, 2).reshape(b, hk, cols * p, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, hk, cols * p, d)
    x = s["q"].float().view(b, q, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    score = torch.matmul(x, k.transpose(-1, -2).contiguous()).view(b, hk, hq // hk, q, cols * p) * s["scale"]
    j = torch.arange(cols * p, device=DEV)
    pos = s["lens"].long()[:, None] - q + torch.arange(q, device=DEV)
    seen = j <= pos[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    w = torch.exp(score - score.amax(-1, keepdim=True))
    w = (w / w.sum(-1, keepdim=True)).view(b, hk, -1, cols * p)
    o = torch.matmul(w, v).view(b, hk, hq // hk, q, d).permute(0, 3, 1, 2, 4)
    return o.reshape(b * q, hq, d).to(s["q"].dtype)


_plain = {"slots": _plain_slots, "rope": _plain_rope, "append": _plain_append, "attn": _plain_attn}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "slots":
        ctx, new = _lengths(case)
        p, n = case["page"], sum(new) + case["pad"]
        fresh = sum(-(-(c + a) // p) - -(-c // p) for c, a in zip(ctx, new))
        return {"bytes": 8 * case["B"] + 8 * fresh + 16 * n + 8 * case["B"], "flops": n}
    hq, hk, d = HEADS[case["heads"]]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "rope":
        t = case["T"]
        return {"bytes": 2 * t * (hq + hk) * d * size + 8 * t, "flops": 3 * t * (hq + hk) * d * case["part"]}
    if case["kind"] == "append":
        t = sum(_lengths(case)[1])
        return {"bytes": 2 * t * hk * d * (size + 1) + 8 * t, "flops": 4 * t * hk * d}
    q, w = case["q"], case["window"] or 1 << 40
    lens = _spread(case["B"], case["lo"], case["hi"])
    tokens = sum(min(n, w + q - 1) for n in lens)
    pairs = sum(min(n - q + 1 + i, w) for n in lens for i in range(q))
    return {"bytes": 2 * tokens * hk * d + 2 * tokens // case["page"] * hk * 4 + 2 * 2 * case["B"] * q * hq * d,
            "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def _e4m3(x):
    """float64 values rounded to the nearest e4m3 number, ties to even (|x| <= 448)."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -7))
    step = _powers(-9, 5).double()[(e - 4).clamp(-9, 5).long() + 9]
    return torch.round(x / step) * step


def _exact_append(s):
    p = s["case"]["page"]
    slots = s["slots"].tolist()
    rows = {}
    for t, slot in enumerate(slots):
        rows.setdefault(slot // p, []).append((t, slot % p))
    r = {n: s[n].double() for n in ("k", "v", "k_scale", "v_scale")}
    for name in ("k", "v"):
        x = s[name + "_new"].double()
        for page, at in rows.items():
            t, row = torch.tensor([a for a, _ in at], device=DEV), torch.tensor([o for _, o in at], device=DEV)
            amax = x[t].abs().amax((0, 2))
            need = torch.full_like(amax, 2.0 ** MAX_EXP)
            for e in range(MAX_EXP - 1, MIN_EXP - 1, -1):  # the smallest power of two that holds amax
                need = torch.where(amax <= F8_MAX * 2.0 ** e, torch.full_like(amax, 2.0 ** e), need)
            old = r[name + "_scale"][page]
            new = need if 0 in [o for _, o in at] else torch.maximum(old, need)
            codes = r[name][page] if name == "k" else r[name][page].transpose(1, 2)  # [hk, p, d]
            if 0 not in [o for _, o in at]:
                codes = torch.where((new > old)[:, None, None], _e4m3(codes * (old / new)[:, None, None]), codes)
            else:
                codes = codes.clone()
            codes[:, row] = _e4m3(x[t].transpose(0, 1) / new[:, None, None])
            r[name][page] = codes if name == "k" else codes.transpose(1, 2)
            r[name + "_scale"][page] = new
    return r


def _exact_attn(s):
    case = s["case"]
    hq, hk, d = HEADS[case["heads"]]
    q, p, group = case["q"], case["page"], hq // hk
    out = torch.zeros(case["B"] * q, hq, d, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_spread(case["B"], case["lo"], case["hi"])):
        low = max(0, n - q - case["window"] + 1) // p if case["window"] else 0
        page = s["table"][b, low:-(-n // p)].long()
        j = torch.arange(low * p, n, device=DEV)
        pos = torch.arange(n - q, n, device=DEV)
        unseen = j[None] > pos[:, None]
        if case["window"]:
            unseen |= j[None] <= pos[:, None] - case["window"]
        for h in range(hk):
            k = (s["k"][page, h].double() * s["k_scale"][page, h].double()[:, None, None]).reshape(-1, d)[:j.numel()]
            v = s["v"][page, h].double() * s["v_scale"][page, h].double()[:, None, None]
            v = v.transpose(1, 2).reshape(-1, d)[:j.numel()]
            for c in range(h * group, (h + 1) * group):
                a = s["q"][b * q:(b + 1) * q, c].double() @ k.t().contiguous() * s["scale"]
                w = torch.softmax(a.masked_fill(unseen, float("-inf")), -1)
                out[b * q:(b + 1) * q, c] = w @ v
    return out


def exact(case, seed):
    if case["kind"] == "slots":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "attn":
        return _exact_attn(s)
    f, r = s["freq"], {}
    n = f.numel()
    first = torch.arange(n, device=DEV) * (2 if case["inter"] else 1)
    second = first + (1 if case["inter"] else n)
    turn = torch.polar(torch.full((case["T"], n), s["mscale"], dtype=torch.float64, device=DEV),
                       s["pos"].double()[:, None] * f)
    for name in ("q", "k"):
        x = s[name].double()
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
        x[..., first], x[..., second] = z.real, z.imag
        r[name] = x
    return r
