"""float64 restatement of the 8-bit paged K/V cache operators (CPU tensors).

``slots`` and ``append`` are exact (whole numbers, codes and scales);
``attention`` and ``rope`` return float64 results, ``attention`` with what an
error bound needs besides.  Written from the definitions in
include/gemmainfer_amd.h, one request, page and row at a time.
"""
from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
MIN_EXP, MAX_EXP, F8_MAX = -40, 40, 448.0


def slots(ctx, new, table, free, used, page, rows):
    """(slots, positions, q_start, seq_lens, status, table) as lists; ``table`` a list of lists."""
    table = [list(r) for r in table]
    cols = len(table[0]) if table else 0
    out, pos, start, lens = [], [], [0], []
    taken = lacking = dropped = 0
    left = max(len(free) - used, 0)
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        fit = min(n, rows - len(out))
        dropped += n - fit
        for j in range(-(-c // page), -(-(c + fit) // page)):
            if j >= cols:
                lacking += 1
                continue
            if taken < left:
                table[b][j] = free[used + taken]
                taken += 1
            else:
                table[b][j] = -1
                lacking += 1
        for p in range(c, c + fit):
            j = p // page
            at = table[b][j] if j < cols else -1
            out.append(at * page + p % page if at >= 0 else -1)
            pos.append(p)
        start.append(len(out))
        lens.append(c + fit)
    pad = rows - len(out)
    return out + [-1] * pad, pos + [0] * pad, start, lens, [used + taken, lacking, dropped], table


def page_scale(amax: float) -> float:
    """The smallest power of two s >= 2^-40 with amax <= 448 s, or NaN."""
    if not math.isfinite(amax) or amax > F8_MAX * 2.0 ** MAX_EXP:
        return math.nan
    e = MIN_EXP
    while amax > F8_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """float64 values (|x| <= 448) rounded to the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -7))
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def append(k, v, slot_list, cache):
    """The cache (CPU tensors k, v, k_scale, v_scale) after the rows k, v are stored; new tensors."""
    kc, vc, ks, vs = [t.clone() for t in cache]
    pages, hk, page, _ = kc.shape
    rows = {}
    for t, s in enumerate(slot_list):
        if 0 <= s < pages * page:
            rows.setdefault(s // page, {})[s % page] = t  # the last row of a slot stays
    for p, at in rows.items():
        place, t = torch.tensor(list(at)), torch.tensor(list(at.values()))
        for x, codes, scale, axis in ((k, kc, ks, 1), (v, vc, vs, 2)):
            for h in range(hk):
                new = x[t, h].double()
                amax = float("nan") if torch.isnan(new).any() else float(new.abs().max())
                need, old = page_scale(amax), float(scale[p, h])
                if 0 in at or math.isnan(need):
                    now = need
                else:
                    now = old if math.isnan(old) or old >= need else need
                held = codes[p, h].double() if axis == 1 else codes[p, h].double().t()
                if 0 not in at and not math.isnan(now) and now > old:
                    held = to_e4m3(held * (old / now))
                held[place] = torch.zeros_like(new) if math.isnan(now) else to_e4m3(new / now)
                codes[p, h] = (held if axis == 1 else held.t()).to(torch.float32).to(E4M3)
                scale[p, h] = now
    return kc, vc, ks, vs


def attention(q, cache, table, lens, starts, scale, window=0):
    """(out, weighted, spread): out float64 [T, Hq, D] (zeros for rows that see nothing, and for
    rows of no request); ``weighted`` = sum_j p_j |v_j|, and ``spread`` [T, Hq, 1] = the largest
    scale * sum_d |q_d k_jd| of a row, the size that errors of its scores are relative to."""
    kc, vc, ks, vs = cache
    _, hk, page, d = kc.shape
    t, hq, _ = q.shape
    group = hq // hk
    out = torch.zeros(t, hq, d, dtype=torch.float64)
    weighted, spread = torch.zeros_like(out), torch.zeros(t, hq, 1, dtype=torch.float64)
    for b, n in enumerate(lens):
        rows = starts[b + 1] - starts[b]
        for i in range(rows):
            row, pos = starts[b] + i, n - rows + i
            low = max(0, pos - window + 1) if window else 0
            if pos < low:
                continue
            j = torch.arange(low, pos + 1)
            at = torch.tensor([int(table[b][c]) for c in range(low // page, pos // page + 1)])
            p = at[j // page - low // page]
            for h in range(hk):
                kk = kc[p, h, j % page].double() * ks[p, h].double()[:, None]
                vv = vc[p, h, :, j % page].double() * vs[p, h].double()[:, None]
                x = q[row, h * group:(h + 1) * group].double()
                w = torch.softmax(x @ kk.t() * scale, -1)
                out[row, h * group:(h + 1) * group] = w @ vv
                weighted[row, h * group:(h + 1) * group] = w @ vv.abs()
                spread[row, h * group:(h + 1) * group, 0] = (x.abs() @ kk.abs().t()).amax(-1) * abs(scale)
    return out, weighted, spread


def rope(x, positions, freq, interleaved, mscale):
    """Rotated float64 [T, H, D], and |x1| + |x2| of each element's pair (0 where it is not rotated)."""
    x = x.double()
    n = freq.numel()
    first = torch.arange(n) * (2 if interleaved else 1)
    second = first + (1 if interleaved else n)
    a = positions.double()[:, None, None] * freq.double()
    x1, x2 = x[..., first], x[..., second]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., first] = mscale * (x1 * a.cos() - x2 * a.sin())
    y[..., second] = mscale * (x2 * a.cos() + x1 * a.sin())
    size[..., first] = size[..., second] = x1.abs() + x2.abs()
    return y, size
