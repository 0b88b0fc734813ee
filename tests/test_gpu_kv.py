"""Slots, rotary rows, append and attention over the 8-bit paged cache, against
the float64 oracle (oracle/kv_oracle.py), at the sizes and masks where they can go wrong."""
import random

import pytest
import torch

from gemmainfer_amd import _lib as L
from gemmainfer_amd import ops, synth
from oracle import kv_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# slots
# ---------------------------------------------------------------------------
def _check_slots(ctx, new, page, rows, cols, n_free, used, pad=0):
    rng = random.Random(len(ctx) * 7 + rows)
    ids = list(range(3, 3 + 4 * (n_free + sum(-(-max(c, 0) // page) for c in ctx)) + 50))
    rng.shuffle(ids)
    table = [[ids.pop() if j < -(-c // page) else -1 for j in range(cols)] for c in ctx]
    free = ids[:n_free]
    wide = torch.full((len(ctx), cols + pad), -7, dtype=torch.int32)
    if ctx and cols:
        wide[:, :cols] = torch.tensor(table, dtype=torch.int32)
    wide = wide.to(DEV)
    free_t, used_t = _i32(free), _i32([used])
    r = ops.kv_slots(_i32(ctx), _i32(new), wide[:, :cols], free_t, used_t, page, rows)
    s, p, start, lens, status, want = O.slots(ctx, new, table, free, used, page, rows)
    assert r.slots.tolist() == s
    assert r.positions.tolist() == p
    assert r.q_start.tolist() == start
    assert r.seq_lens.tolist() == lens
    assert r.status.tolist() == status
    assert wide[:, :cols].tolist() == want
    assert (wide[:, cols:] == -7).all()
    assert free_t.tolist() == free and used_t.tolist() == [used]


@pytest.mark.parametrize("b,page", [(1, 16), (3, 32), (64, 16), (257, 64), (1000, 256)])
def test_slots_ragged(b, page):
    rng = random.Random(b)
    ctx = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, 900)]) for _ in range(b)]
    new = [rng.choice([0, 1, 1, page, page + 1, rng.randint(0, 70)]) for _ in range(b)]
    need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(ctx, new))
    cols = max(-(-(c + n) // page) for c, n in zip(ctx, new)) + 1
    _check_slots(ctx, new, page, sum(new) + 5, cols, need + 4, 2, pad=3)


@pytest.mark.parametrize("ctx,new,rows,cols,n_free,used", [
    ([], [], 0, 4, 3, 0),                              # no requests, no rows
    ([], [], 300, 0, 0, 0),                            # only padding
    ([5, 9], [0, 0], 7, 2, 1, 0),                      # nothing to add
    ([0, 0, 16], [40, 1, 1], 20, 4, 9, 0),             # rows dropped inside a request
    ([0, 30, 16], [40, 10, 30], 80, 4, 2, 0),          # the list runs out inside a request
    ([0, 30], [40, 10], 50, 4, 2, 2),                  # none left
    ([0, 30], [40, 10], 50, 4, 2, 9),                  # more used than there are
    ([0, 30], [200, 10], 210, 4, 40, 1),               # a request longer than its table
    ([70], [3], 3, 4, 5, 0),                           # ... already before the step
    ([-4, 3], [5, -2], 9, 2, 3, 0),                    # negative lengths count as none
    ([0], [5000], 5000, 320, 313, 0),                  # one prompt over many workgroups
])
def test_slots_edges(ctx, new, rows, cols, n_free, used):
    _check_slots(ctx, new, 16, rows, cols, n_free, used)


def test_slots_many_requests_and_status_chain():
    b = 8192
    table = torch.full((b, 3), -1, dtype=torch.int32, device=DEV)
    free = torch.arange(2 * b, dtype=torch.int32, device=DEV)
    one = torch.ones(b, dtype=torch.int32, device=DEV)
    r = ops.kv_slots(torch.zeros_like(one), one, table, free, _i32([0]), 16, b)
    assert torch.equal(r.slots, torch.arange(b, device=DEV) * 16)
    r = ops.kv_slots(r.seq_lens, 15 * one, table, free, r.status, 16, 15 * b)
    assert r.status.tolist() == [b, 0, 0]
    r = ops.kv_slots(r.seq_lens, one, table, free, r.status, 16, b)
    assert r.status.tolist() == [2 * b, 0, 0]
    assert torch.equal(r.slots, (torch.arange(b, device=DEV) + b) * 16)
    r = ops.kv_slots(r.seq_lens, 16 * one, table, free, r.status, 16, 16 * b)
    assert r.status.tolist() == [2 * b, b, 0]          # the last of each request's 16 rows has no page
    assert (r.slots.view(b, 16)[:, 15] == -1).all() and (r.slots.view(b, 16)[:, :15] >= 0).all()


# ---------------------------------------------------------------------------
# rope
# ---------------------------------------------------------------------------
HALF = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}  # half a step, relative (finfo.eps / 2)


def _check_rope(got, x, pos, freq, inter, mscale):
    # the reduced angle is off by 2^-26 turns (4.7e-8 rad half step, 9.4e-8 with the fp64 product's
    # rounding at these positions), cos and sin by a few units of 2^-24, two products and a sum by three
    # roundings: under 2^-20 (9.5e-7) of |x1| + |x2| together, then half a step of the stored type
    y, size = O.rope(x, pos, freq, inter, mscale)
    bound = HALF[x.dtype] * y.abs() + 2.0 ** -20 * mscale * size
    bound += (2.0 ** -25 if x.dtype == FP16 else 0.0)  # fp16's subnormal half step
    assert ((got.double() - y).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("t,hq,hk,d,rot,inter", [
    (1, 16, 2, 512, 128, False), (3, 4, 1, 64, 64, True), (257, 16, 8, 256, 256, False), (5, 3, 3, 128, 48, True),
    (7, 2, 1, 80, 40, False), (2, 5, 2, 30, 6, True), (4, 1, 1, 66, 66, False), (2, 1, 1, 1024, 1024, True),
    (6, 2, 2, 64, 24, True), (6, 2, 2, 64, 24, False)])
def test_rope_rows(dtype, t, hq, hk, d, rot, inter):
    g = _gen(t * d)
    q, k = torch.randn(t, hq, d, generator=g).to(dtype), torch.randn(t, hk, d, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (t,), generator=g)
    freq, mscale = ops.rope_frequencies(rot, 1e4, scaling="yarn", factor=4.0, device=DEV)
    qd, kd = q.to(DEV), k.to(DEV)
    qo, ko = ops.rope_rows(qd, kd, pos.to(DEV), freq, interleaved=inter, mscale=mscale)
    assert torch.equal(qd.cpu(), q) and torch.equal(kd.cpu(), k)
    _check_rope(qo.cpu(), q, pos, freq.cpu(), inter, mscale)
    _check_rope(ko.cpu(), k, pos, freq.cpu(), inter, mscale)
    # in place, on slices of a wider tensor: the same bits, and nothing around them
    wide = torch.full((t, hq + hk + 1, d + 8), 3.0, dtype=dtype, device=DEV)
    qs, ks = wide[:, :hq, :d], wide[:, hq:hq + hk, :d]
    qs.copy_(qd), ks.copy_(kd)
    a, b = ops.rope_rows(qs, ks, pos.to(DEV), freq, interleaved=inter, mscale=mscale, inplace=True)
    assert a is qs and b is ks
    assert torch.equal(qs, qo) and torch.equal(ks, ko)
    assert (wide[:, hq + hk:] == 3).all() and (wide[..., d:] == 3).all()
    # heads before rows, an odd offset, no k
    buf = torch.empty(hq * t * d + 1, dtype=dtype, device=DEV)[1:].view(hq, t, d).transpose(0, 1)
    buf.copy_(qd)
    only, none = ops.rope_rows(buf, None, pos.to(DEV), freq, interleaved=inter, mscale=mscale)
    assert none is None and torch.equal(only, qo)


def test_rope_more_rows_than_a_grid_is_wide():
    """2^24 rows and more: the last ones turn as they do in a call of their own."""
    t, n, d = (1 << 24) + 300, 500, 16
    freq, _ = ops.rope_frequencies(d, device=DEV)
    q = torch.zeros(t, 1, d, dtype=BF16, device=DEV)
    pos = torch.zeros(t, dtype=torch.int64, device=DEV)
    own = torch.randn(n, 1, d, generator=_gen(1)).to(BF16).to(DEV)
    ats = (0, (1 << 23) - 250, t - n)
    for at in ats:
        q[at:at + n] = own
        pos[at:at + n] = torch.arange(n, device=DEV)
    want, _ = ops.rope_rows(q[:n], None, pos[:n], freq)
    got, _ = ops.rope_rows(q, None, pos, freq)
    assert torch.equal(got, ops.rope_rows(q, None, pos, freq, inplace=True)[0])
    assert not got[n:ats[1]].any() and not got[ats[1] + n:ats[2]].any()
    for at in ats:
        assert torch.equal(got[at:at + n], want)


def test_rope_matches_the_table_form():
    """fused_rope_inplace with tables of the same angles: equal to a rounding of each."""
    t, d = 33, 256
    q = torch.randn(t, 4, d, generator=_gen(1)).to(DEV)
    freq, _ = ops.rope_frequencies(d, device=DEV)
    ang = torch.arange(t, device=DEV, dtype=torch.float64)[:, None] * freq
    ang = torch.cat([ang, ang], -1)
    ref = q.transpose(0, 1)[None].clone()
    ops.fused_rope_inplace(ref, None, ang.cos().float(), ang.sin().float(), torch.arange(t, device=DEV)[None])
    out, _ = ops.rope_rows(q, None, torch.arange(t, device=DEV), freq)
    assert ((ref[0].transpose(0, 1) - out).abs() <= 2.0 ** -19 * (q.abs() + q.abs().roll(d // 2, -1))).all()


def test_rope_empty_and_negative_positions():
    freq, _ = ops.rope_frequencies(64, device=DEV)
    e = torch.empty(0, 2, 64, dtype=BF16, device=DEV)
    assert ops.rope_rows(e, e, torch.empty(0, dtype=torch.int64, device=DEV), freq)[0].shape == (0, 2, 64)
    q, pos = torch.randn(3, 2, 64, generator=_gen(2)), torch.tensor([-5, 0, -100000])
    got, _ = ops.rope_rows(q.to(DEV), None, pos.to(DEV), freq)
    _check_rope(got.cpu(), q, pos, freq.cpu(), False, 1.0)


def test_rope_frequency_scaling():
    base, _ = ops.rope_frequencies(128, 5e5, device="cpu")
    lin, m = ops.rope_frequencies(128, 5e5, scaling="linear", factor=8, device="cpu")
    assert torch.equal(lin, base / 8) and m == 1.0
    ntk, _ = ops.rope_frequencies(128, 5e5, scaling="ntk", factor=8, device="cpu")
    assert ntk[0] == 1 and abs(float(ntk[-1] / base[-1]) - 1 / 8) < 1e-12
    yarn, m = ops.rope_frequencies(128, 5e5, scaling="yarn", factor=8, original_len=4096, device="cpu")
    turns = 4096 * base / (2 * torch.pi)
    assert torch.equal(yarn[turns > 32], base[turns > 32])
    assert torch.allclose(yarn[turns < 1], base[turns < 1] / 8, rtol=1e-15, atol=0) and m > 1


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _filled(pages, hk, page, d, seed, spread=1.0):
    """A cache (CPU tensors) of random pages whose sizes differ by page and head."""
    g = _gen(seed)
    r = []
    for shape in ((pages, hk, page, d), (pages, hk, d, page)):
        x = torch.randn(shape, generator=g) * torch.exp2(spread * torch.randn(pages, hk, 1, 1, generator=g))
        s = torch.tensor([[O.page_scale(float(x[p, h].abs().max())) for h in range(hk)] for p in range(pages)])
        r.append(((x / s[:, :, None, None]).to(O.E4M3), s))
    return ops.KVCache(r[0][0], r[1][0], r[0][1], r[1][1])


def _to(cache, dev):
    return ops.KVCache(*[t.to(dev).clone() for t in cache])


def _same_cache(got, want):
    for name, x, y in zip(got._fields, got, want):
        x = x.cpu()
        if x.dtype == O.E4M3:
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), name
        else:
            assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x[~torch.isnan(x)], y[~torch.isnan(y)]), name


def _check_append(cache, k, v, slots):
    dev = _to(cache, DEV)
    ops.kv_append(k.to(DEV), v.to(DEV), torch.tensor(slots, dtype=torch.int64, device=DEV), dev)
    want = O.append(k, v, slots, cache)
    _same_cache(dev, want)
    return ops.KVCache(*want)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("page,d,hk", [(16, 64, 1), (32, 128, 3), (64, 256, 2), (128, 512, 1), (256, 64, 2)])
def test_append_runs(dtype, page, d, hk):
    """Rows into the middle of pages, over page ends, whole pages, lone rows; small rows and ones
    that raise the scale; then the same call again changes nothing."""
    pages = 9
    cache = _filled(pages, hk, page, d, seed=page)
    g = _gen(d)
    slots = [3 * page + page - 2, 3 * page + page - 1, *range(5 * page, 6 * page), 7 * page, 7 * page + 1,
             *range(1 * page + 5, 1 * page + page - 1), 8 * page + 3, 2 * page + page // 2]
    t = len(slots)
    size = torch.exp2(2 * torch.randn(t, hk, 1, generator=g))
    k = (torch.randn(t, hk, d, generator=g) * size).to(dtype)
    v = (torch.randn(t, hk, d, generator=g) * size).to(dtype)
    once = _check_append(cache, k, v, slots)
    again = _check_append(once, k, v, slots)
    _same_cache(_to(again, "cpu"), once)


@pytest.mark.parametrize("t,hk,page", [(1, 1, 16), (700, 2, 16), (300, 40, 64)])
def test_append_prompt_and_decode_sized_grids(t, hk, page):
    """Both grid forms (a workgroup for each row, for sixteen rows), and runs cut by their borders."""
    pages = -(-t // page) + 3
    cache = ops.KVCache(*[x.cpu() for x in ops.kv_cache(pages, hk, page, 64, DEV)])
    k, v = torch.randn(t, hk, 64, generator=_gen(t)).to(BF16), torch.randn(t, hk, 64, generator=_gen(t + 1)).to(BF16)
    first = [2 * page + i for i in range(t)]
    cache = _check_append(cache, k, v, first)
    n = max(1, t // 2)
    _check_append(cache, 3 * k[:n], 3 * v[:n], [s + 5 for s in first[:n]])


def test_append_skips_duplicates_and_bad_slots():
    page, d = 16, 64
    cache = _filled(6, 2, page, d, seed=4)
    slots = [-1, -5, 17, 18, 17, 17, -1, 6 * page, 6 * page + 3, 1 << 40, 33, 33, 33, -(1 << 40), 95, -1]
    k = torch.randn(len(slots), 2, d, generator=_gen(1)).to(BF16)
    k[3] *= 300  # the larger of two rows that go to different places
    k[2] *= 1e6  # a row that another one replaces: it does not count
    _check_append(cache, k, k.flip(0), slots)
    # padding that names place 0 over and over: one row stays
    _check_append(cache, k, k.flip(0), [0] * len(slots))
    many = torch.randn(900, 2, d, generator=_gen(2)).to(BF16)
    _check_append(cache, many, many, [3 * page + i % 5 for i in range(900)])
    e = torch.empty(0, 2, d, dtype=BF16)
    _check_append(cache, e, e, [])


def _sized_rows(t, hk, d, seed):
    """Rows whose sizes differ by powers of two, so that rows all along a run raise its page's scale."""
    g = _gen(seed)
    size = torch.exp2(3 * torch.randn(t, hk, 1, generator=g))
    return ((torch.randn(t, hk, d, generator=g) * size).to(BF16) for _ in range(2))


@pytest.mark.parametrize("hk", [2, 700])
def test_append_skipped_rows_inside_a_page(hk):
    """Rows of one page with skipped ones between them are one run: the page's scale is that of them
    all, whichever raises it.  2 heads: a workgroup a row; 700: sixteen rows a workgroup."""
    page, pages = 16, 5
    cache = _filled(pages, hk, page, 8, seed=hk)
    for slots in ([17, -1, 18], [-1, 17, -1, -9, 18, -1], [17, pages * page, 1 << 40, 18, -(1 << 40), 19],
                  [20, -1, 33, -1, 34, -1, 48, -1, 49, -1], [-1, -1, 18, 19, -1, 20, -1, -1, 21, 36, -1, 37, -1, 38, 70, -1]):
        slots = slots + [-1] * (16 - len(slots))
        n = len(slots)
        rows = torch.exp2(torch.arange(n).float() * 2 - 6).view(n, 1, 1) * torch.ones(n, hk, 8)
        _check_append(cache, rows.to(BF16), rows.flip(0).to(BF16), slots)
        k, v = _sized_rows(n, hk, 8, n)
        _check_append(cache, k, v, slots)


@pytest.mark.parametrize("hk", [1, 40])
@pytest.mark.parametrize("hole", [14, 15, 16, 47, 48, 62, 63, 64, 65, 255, 256, 257, 511, 512, 513, 575, 576, 2303, 2304,
                                  2305, 5000])
def test_append_holes_of_any_length(hk, hole):
    """Skipped rows before, between and behind the rows of a page, over every number of rows that is
    looked at together."""
    page = 16
    cache = _filled(6, hk, page, 8, seed=hole)
    for slots in ([17] + [-1] * hole + [18, 19, 35],                              # one page on both sides
                  [17] + [-1] * hole + [33, 34] + [6 * page] * hole + [35],      # another behind it, then one again
                  [-1] * hole + [49] + [-1] * hole):
        k, v = _sized_rows(len(slots), hk, 8, hole)
        _check_append(cache, k, v, slots)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("t,hk", [(1040, 8), (300, 40), (9000, 1)])
def test_append_many_pages_a_workgroup(t, hk, page):
    """More than 8192 rows of heads, as of a large decode step: lone rows on pages of their own, then
    runs of 3 to 7, whole pages, and skipped rows, so that a workgroup's sixteen rows are many runs."""
    rng = random.Random(t)
    pages = t
    cache = _filled(1, 2, page, 8, seed=t)
    scale = torch.exp2(torch.randint(-8, 3, (2, pages, hk), generator=_gen(t)).float())
    cache = ops.KVCache(cache.k.view(torch.uint8)[:, :1].expand(pages, hk, page, 8).contiguous().view(O.E4M3),
                        cache.v.view(torch.uint8)[:, 1:].expand(pages, hk, 8, page).contiguous().view(O.E4M3),
                        scale[0].contiguous(), scale[1].contiguous())
    for runs in ([1], [1, 3, 7, 4], [1, 2, 5, page, 2 * page]):
        ids = list(range(pages))
        rng.shuffle(ids)
        slots = []
        while len(slots) < t:
            n, p = rng.choice(runs), ids.pop()
            first = rng.randrange(page)
            slots += [p * page + (first + i) % page for i in range(n)]
            if rng.random() < 0.2:
                slots.append(rng.choice([-1, pages * page + 5]))
        k, v = _sized_rows(t, hk, 8, t)
        _check_append(cache, k, v, slots[:t])


@pytest.mark.parametrize("page,hk,t", [(16, 2, 900), (16, 40, 900), (64, 40, 2000), (256, 33, 1500)])
def test_append_random_runs_and_holes(page, hk, t):
    """Pages in any order, runs of 1 to 40 rows in any order of places (some named twice), holes of
    1 to 90 rows anywhere."""
    rng = random.Random(page * hk)
    pages = 700
    ids = list(range(pages))
    rng.shuffle(ids)
    slots = []
    while len(slots) < t:
        p = ids.pop()
        for _ in range(rng.choice([1, 1, 1, 2, 7, 16, 40])):
            slots.append(p * page + rng.randrange(page))
            if rng.random() < 0.1:
                slots += [-1] * rng.choice([1, 1, 2, 15, 90])
        slots += [-1] * rng.choice([0, 0, 0, 1, 5, 70])
    cache = _filled(pages, 2, page, 8, seed=page)
    cache = ops.KVCache(*[x.repeat_interleave(-(-hk // 2), 1)[:, :hk].contiguous() if x.dtype == FP32 else
                          x.view(torch.uint8).repeat_interleave(-(-hk // 2), 1)[:, :hk].contiguous().view(O.E4M3)
                          for x in cache])
    k, v = _sized_rows(len(slots), hk, 8, t)
    _check_append(cache, k, v, slots)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), 3e38, 448.0 * 2 ** 40, 2.0 ** -133, 0.0])
def test_append_extreme_values(value):
    page, d = 16, 64
    cache = _filled(4, 2, page, d, seed=6)
    k, v = torch.randn(3, 2, d, generator=_gen(3)).to(BF16), torch.zeros(3, 2, d, dtype=BF16)
    k[1, 1, 7] = v[2, 0, 3] = value
    cache = _check_append(cache, k, v, [17, 18, 40])
    # a page without a scale keeps none while it is added to ...
    cache = _check_append(cache, torch.ones_like(k), torch.ones_like(k), [19, 20, 41])
    # ... until its first place is written
    cache = _check_append(cache, torch.ones_like(k), torch.ones_like(k), [16, 17, 32])
    assert not torch.isnan(cache.k_scale).any() and not torch.isnan(cache.v_scale).any()


def test_append_rounds_and_rescales_every_code():
    """Every e4m3 code moves to scales 1, 2, 4, ... 512 times as large, and every border between
    two codes is rounded, as the definition says."""
    page, d = 32, 256
    codes = torch.arange(256, dtype=torch.uint8)
    codes[127] = codes[255] = 0  # NaN codes are never written
    cache = ops.KVCache(*[x.cpu() for x in ops.kv_cache(12, 1, page, d, DEV)])
    cache.k.view(torch.uint8)[:, 0, 3] = codes
    cache.v.view(torch.uint8)[:, 0, :, 3] = codes
    cache.k_scale.fill_(2.0), cache.v_scale.fill_(0.25)
    for e in range(11):
        x = torch.zeros(1, 1, d, dtype=FP32)
        x[0, 0, 0] = 448.0 * 2 ** e
        _check_append(cache, x, x, [e * page + 9])
    values = torch.unique(codes.view(O.E4M3).double())
    mid = (values[1:] + values[:-1]) / 2
    x = torch.cat([mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), values, values[:4]]).float()
    x = torch.cat([x, torch.zeros(-len(x) % d)]).view(-1, 1, d)
    x[:, 0, -1] = 448.0
    _check_append(cache, x, x, list(range(2 * page, 2 * page + x.shape[0])))


def test_append_more_rows_than_a_grid_is_wide():
    """2^28 rows and more, 2^20 to a page: of each place the last one stays."""
    t, group, page, d = (1 << 28) + (1 << 20) + 5, 1 << 20, 16, 8
    row = torch.arange(t, device=DEV)
    slots = row // group * page + row % page
    x = torch.empty(t, 1, d, dtype=BF16, device=DEV)
    x[:] = (row % 1009).to(BF16)[:, None, None]
    pages = t // group + 1
    cache, want = ops.kv_cache(pages, 1, page, d * 8, DEV), ops.kv_cache(pages, 1, page, d * 8, DEV)
    cache, want = (c._replace(k=c.k[..., :d].contiguous(), v=c.v[:, :, :d].contiguous()) for c in (cache, want))
    ops.kv_append(x, -x, slots, cache)
    ends = [min((p + 1) * group, t) for p in range(pages)]
    last = torch.cat([torch.arange(max(e - page, p * group), e) for p, e in enumerate(ends)]).to(DEV)
    assert pages == 258 and last.numel() == 257 * page + 5
    ops.kv_append(x[last], -x[last], slots[last], want)
    for a, b in zip(cache, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_strided_rows():
    page, d, hk, t = 16, 128, 2, 21
    cache = _filled(5, hk, page, d, seed=8)
    qkv = torch.randn(t, 7 * d + 3, generator=_gen(5)).to(BF16)
    slots = list(range(page + 3, page + 3 + t))
    want = O.append(qkv[:, 3 * d:5 * d].reshape(t, hk, d), qkv[:, 5 * d + 3:7 * d + 3].reshape(t, hk, d), slots, cache)
    on = qkv.to(DEV)
    dev = _to(cache, DEV)
    s = torch.tensor(slots, device=DEV)
    ops.kv_append(on[:, 3 * d:5 * d].unflatten(1, (hk, d)), on[:, 5 * d + 3:].unflatten(1, (hk, d)), s, dev)
    _same_cache(dev, want)
    # heads before rows
    dev = _to(cache, DEV)
    k, v = on[:, 3 * d:5 * d].unflatten(1, (hk, d)), on[:, 5 * d + 3:].unflatten(1, (hk, d))
    ops.kv_append(k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(0, 1).contiguous().transpose(0, 1), s, dev)
    _same_cache(dev, want)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _setup(lens, rows, hk, page, d, seed, spread=1.0, extra=2):
    """A cache on the CPU, its table (entries behind a request's pages lead nowhere), q_start."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra
    cache = _filled(pages, hk, page, d, seed, spread)
    ids = list(range(pages))
    random.Random(seed).shuffle(ids)
    cols = max(need, default=0) + 1
    table = [[ids.pop() if c < n else -1 for c in range(cols)] for n in need]
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    return cache, table, start


def _check_out(got, ref, weighted, spread, d, tokens):
    """Errors of the kernel: a score is an fp32 sum of D exact products and three more roundings, in
    the exponent's unit (1/ln 2) beside log2 of a scale (|.| <= 40): e = (D + 8) 2^-24 (spread + 28); weights
    are rounded to fp16 as 8 = 2^3 times their share of a weight that is no larger than the largest
    (half a step is 2^-11 of it down to fp16's 2^-14, so of a weight over 2^-17; below that 2^-25,
    2^-28 of that weight, and twice that with the weight's own sum) and so
    are off by w = 2^-11 + 2 e together with the fp32 sums of the weights (tokens 2^-24, and of the
    products: the same); the result is stored in half a step."""
    e = (d + 8) * 2.0 ** -24 * (spread + 28)
    w = 2.0 ** -11 + 2 * e + 2 * tokens * 2.0 ** -24
    bound = HALF[got.dtype] * ref.abs() + (1 + HALF[got.dtype]) * w * weighted + tokens * 2.0 ** -27 * weighted.amax()
    bound += 2.0 ** -24 if got.dtype == FP16 else 0.0
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"{(err - bound).max()} over, {(err / bound.clamp(min=1e-30)).max()} of the bound"


def _check_attention(lens, rows, hq, hk, page, d, dtype, window=0, seed=0, decode=False, scale=None, spread=1.0,
                     q_size=2.0):
    cache, table, start = _setup(lens, rows, hk, page, d, seed, spread)
    q = (q_size * torch.randn(start[-1], hq, d, generator=_gen(seed + 1))).to(dtype)
    dev = _to(cache, DEV)
    got = ops.kv_attention(q.to(DEV), dev, _i32(table), _i32(lens), None if decode else _i32(start), scale=scale,
                           window=window)
    ref, weighted, size = O.attention(q, cache, table, lens, start, d ** -0.5 if scale is None else scale, window)
    _check_out(got, ref, weighted, size, d, max(lens))
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hk,d,page", [(16, 8, 256, 16), (16, 2, 512, 64), (32, 8, 128, 32), (12, 4, 64, 128),
                                          (7, 1, 64, 256), (5, 5, 128, 16), (40, 1, 256, 64)])
def test_attention_decode(dtype, hq, hk, d, page):
    """One row a request: every length around a group of 16, a unit of 64, a page; a long one beside."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 255, 257, 1000, 0, 333]
    _check_attention(lens, [1] * len(lens), hq, hk, page, d, dtype, seed=d + page, decode=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hk,d,page", [(16, 8, 256, 16), (16, 2, 512, 32), (8, 2, 128, 64), (3, 1, 64, 16)])
@pytest.mark.parametrize("window", [0, 1, 17, 64, 100])
def test_attention_ragged_rows(dtype, hq, hk, d, page, window):
    """Prompts, chunks onto a context, verify rows, no rows, rows that see nothing, with windows."""
    lens = [40, 300, 7, 64, 0, 129, 3, 90]
    rows = [40, 33, 7, 1, 0, 8, 5, 0]
    got = _check_attention(lens, rows, hq, hk, page, d, dtype, window, seed=window + d)
    assert (got[40 + 33 + 7 + 1 + 8:40 + 33 + 7 + 1 + 8 + 2] == 0).all()  # request of 3 tokens, 5 rows


@pytest.mark.parametrize("rows,hq,hk,d", [(3, 16, 8, 256), (10, 16, 8, 256), (40, 16, 8, 256), (5, 16, 2, 512),
                                          (20, 16, 2, 512), (70, 4, 4, 64), (30, 4, 4, 128), (100, 4, 4, 128)])
def test_attention_row_tiles(rows, hq, hk, d):
    """Each count of column tiles, cut and whole."""
    _check_attention([rows + 111, rows], [rows, rows], hq, hk, 32, d, BF16, seed=rows)


@pytest.mark.parametrize("b", [64, 65, 130, 300, 4100])
def test_attention_many_requests(b):
    rng = random.Random(b)
    lens = [rng.choice([0, 1, 5, 60, 100]) for _ in range(b)]
    _check_attention(lens, [1] * b, 2, 1, 16, 64, BF16, seed=b, decode=True)
    rows = [rng.choice([0, 1, 2]) for _ in range(b)]
    _check_attention([n + r for n, r in zip(lens, rows)], rows, 2, 1, 16, 64, BF16, seed=b)


@pytest.mark.parametrize("cols", [1, 20])
def test_attention_more_items_than_a_grid_is_wide(cols):
    """2^18 requests on 64 kv heads (2^24 items) against the calls of their 13 x 7 x 17 kinds (row, page, length)."""
    b, hk, d, page = 1 << 18, 64, 64, 16
    cache = _to(_filled(7, hk, page, d, seed=1), DEV)
    q = torch.randn(13, hk, d, generator=_gen(2)).to(BF16).to(DEV)
    kind = torch.arange(13 * 7 * 17, device=DEV)
    pick = torch.randint(0, len(kind), (b,), generator=_gen(3)).to(DEV)
    pick[-len(kind):] = kind

    def call(k):
        table = torch.full((len(k), cols), -1, dtype=torch.int32, device=DEV)
        table[:, 0] = k // 17 % 7
        return ops.kv_attention(q[k // (17 * 7)], cache, table, (k % 17).int())
    want = torch.cat([call(kind[i:i + 60]) for i in range(0, len(kind), 60)])
    got = call(pick)
    for i in range(0, b, 1 << 14):
        assert torch.equal(got[i:i + (1 << 14)], want[pick[i:i + (1 << 14)]])


def test_attention_long_request_among_many():
    """A request over many workgroups beside 99 short ones: its partial sums are where the join looks."""
    lens = [30] * 100
    lens[37] = 20000
    _check_attention(lens, [1] * 100, 8, 2, 64, 64, BF16, seed=8, decode=True, spread=2.0)
    _check_attention(lens, [3] * 100, 8, 2, 64, 64, FP16, seed=9)


@pytest.mark.parametrize("hq,hk,d,rows", [(16, 8, 256, 1), (16, 2, 512, 1), (4, 2, 64, 3), (8, 1, 128, 40)])
def test_attention_long_axis_is_cut_and_joined(hq, hk, d, rows):
    """A context over many workgroups: their partial sums, with sizes that differ from page to page."""
    _check_attention([9001], [rows], hq, hk, 64, d, BF16, seed=rows, spread=3.0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hk,d,page", [(16, 8, 256, 16), (16, 2, 512, 64), (4, 4, 64, 16), (8, 1, 128, 128)])
@pytest.mark.parametrize("window", [512, 1024, 1500])
@pytest.mark.parametrize("lens,rows", [([9000, 1500, 511, 1023], [1, 1, 1, 1]),        # decode
                                       ([1500, 4001, 600, 1030], [7, 1, 5, 7]),        # verify
                                       ([1100, 3000, 40], [130, 33, 40])])             # prompts over the window's end
def test_attention_windowed_requests_are_cut(dtype, hq, hk, d, page, window, lens, rows):
    """Windows of several chunks that start inside the request: partial sums, and the chunks that a
    tile of the list has and its window does not."""
    _check_attention(lens, rows, hq, hk, page, d, dtype, window, seed=window + sum(rows), spread=2.0)


@pytest.mark.parametrize("b", [65, 130])
@pytest.mark.parametrize("hq,hk,d,rows", [(8, 2, 64, 6), (8, 2, 64, 12), (16, 8, 256, 9), (16, 8, 256, 17), (16, 2, 512, 3)])
@pytest.mark.parametrize("window", [0, 512])
def test_attention_many_requests_of_many_rows(b, hq, hk, d, rows, window):
    """The plan of more than 64 requests with tiles of 32 and 64 columns, one request cut and joined,
    some without rows or tokens."""
    rng = random.Random(b * rows)
    counts = [rng.choice([rows, rows, rows, 2 * rows, 1, 0]) for _ in range(b)]
    while sum(counts) < (rows - 1) * b:  # the mean decides the tile
        counts[rng.randrange(b)] = 2 * rows
    lens = [max(0, n + rng.choice([-1, 0, 0, 5, 60])) for n in counts]
    lens[b // 2], counts[b // 2] = 4000, rows
    _check_attention(lens, counts, hq, hk, 16, d, BF16, window, seed=b + rows, spread=2.0)


@pytest.mark.parametrize("hq,hk,d", [(16, 8, 256), (16, 2, 512), (12, 4, 64)])
def test_attention_on_one_workspace(hq, hk, d):
    """The C entry with a workspace for 64 rows of 64 requests: every smaller call is served by it,
    with the bits of a call with its own, and nothing behind it is written."""
    lib, page, n = L.load(), 16, 2000
    cols = n // page
    cache = _to(_filled(cols, hk, page, d, seed=1), DEV)
    table = _i32([list(range(cols))] * 64)
    nbytes = lib.gi_kv_attention_workspace_bytes(64, 64, hq, hk, d, n)
    for t, b in ((64, 64), (64, 1), (64, 2), (64, 3), (64, 4), (64, 9), (40, 2), (17, 1), (9, 1), (1, 1), (5, 64)):
        q = torch.randn(t, hq, d, generator=_gen(t)).to(BF16).to(DEV)
        start = _i32([min(i * -(-t // b), t) for i in range(b + 1)])
        lens = _i32([n - 37 * i % 900 for i in range(b)])
        want = ops.kv_attention(q, cache, table[:b], lens, start)
        ws = torch.full((nbytes + 4096,), 0xAB, dtype=torch.uint8, device=DEV)
        out = torch.zeros_like(q)
        st = lib.gi_kv_attention(q.data_ptr(), L.DTYPE_BF16, hq * d, d, *[x.data_ptr() for x in cache], table.data_ptr(),
                                 cols, cols, lens.data_ptr(), start.data_ptr(), out.data_ptr(), hq * d, d, t, b, hq, hk,
                                 d, page, cols, d ** -0.5, 0, ws.data_ptr(), nbytes,
                                 torch.cuda.current_stream().cuda_stream)
        assert st == L.GI_OK, (t, b, lib.gi_last_error())
        assert torch.equal(out, want) and (ws[nbytes:] == 0xAB).all(), (t, b)


@pytest.mark.parametrize("hk,d,g", [(1, 64, 3), (8, 64, 2), (2, 128, 4), (8, 256, 2), (2, 512, 8)])
def test_attention_partial_sums_have_room(hk, d, g):
    """Batches whose lengths and rows differ by powers of two: no tile is without room for its chunks
    (it would be NaN)."""
    rng = random.Random(d + hk)
    page, cols = 64, 400
    cache = _to(_filled(8, hk, page, d, seed=1), DEV)
    cache = ops.KVCache(*[x[torch.arange(cols, device=DEV) % 8] if x.dtype == FP32 else
                          x.view(torch.uint8)[torch.arange(cols, device=DEV) % 8].view(x.dtype) for x in cache])
    for _ in range(40):
        b = rng.choice([1, 2, 5, 20, 64, 65, 150])
        rows = [int(2 ** rng.uniform(0, rng.choice([0, 3, 6]))) for _ in range(b)]
        lens = [r + int(2 ** rng.uniform(0, rng.choice([6, 10, 14.5]))) for r in rows]
        start = [0]
        for r in rows:
            start.append(start[-1] + r)
        q = torch.randn(start[-1], hk * g, d, generator=_gen(b)).to(BF16).to(DEV)
        got = ops.kv_attention(q, cache, _i32([list(range(cols))] * b), _i32(lens), _i32(start),
                               window=rng.choice([0, 0, 700]))
        assert torch.isfinite(got).all(), (rows, lens)


@pytest.mark.parametrize("window", [0, 50])
def test_attention_peaked_and_flat(window):
    """Weights of one token, scores that run away late, and a scale of 0 (plain means)."""
    for scale, size in ((1.0, 8.0), (0.0, 1.0), (-0.5, 2.0)):
        _check_attention([500, 77], [5, 3], 4, 2, 16, 128, FP16, window, seed=3, scale=scale, q_size=size)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("at", [0, 5, 4000, 8191])
def test_attention_flat_tail_behind_a_heavy_token(dtype, at):
    """One token of 2^30 times the weight of each of 8191 others, with values of its own in half the
    dimensions only: what the others add up to in the rest is seen.  Forty requests, so that a
    request is not cut into chunks, and a wave meets a quarter of it."""
    hk, d, n, b, page = 64, 64, 8192, 40, 64
    g = _gen(at)
    k, v = torch.zeros(n, hk, d), 0.5 + 0.5 * torch.rand(n, hk, d, generator=g)
    k[..., 0] = 2 * torch.rand(n, hk, generator=g) - 1
    k[at, :, 0] = 30.0
    v[at, :, :32], v[at, :, 32:] = 1.5, 0.0
    k, v = k.to(O.E4M3), v.to(O.E4M3)
    ones = torch.ones(n // page, hk)
    cache = ops.KVCache(k.view(n // page, page, hk, d).transpose(1, 2).contiguous(),
                        v.view(n // page, page, hk, d).permute(0, 2, 3, 1).contiguous(), ones, ones)
    q = torch.zeros(b, hk, d)
    q[..., 0] = 16 * torch.exp2(-torch.rand(b, 1, generator=g) / 16)
    q[..., 1:] = torch.randn(b, hk, d - 1, generator=g)
    q = q.to(dtype)
    scale = 0.6931471805599453 / 16
    got = ops.kv_attention(q.to(DEV), _to(cache, DEV), _i32([list(range(n // page))] * b), _i32([n] * b), scale=scale)
    ref, weighted = torch.zeros(b, hk, d, dtype=torch.float64), torch.zeros(b, hk, d, dtype=torch.float64)
    for h in range(hk):
        p = torch.softmax(q[:, h].double() @ k[:, h].double().t() * scale, -1)
        ref[:, h] = weighted[:, h] = p @ v[:, h].double()  # no value is negative
    # as in _check_out, with weights of 2^11 times their share (65504 at most, so the heaviest is 2^11 or more):
    # half a step is 2^-11 of one over 2^-25 of the heaviest, below that 2^-36 of the heaviest, and as much
    # again where the heaviest is up to twice the reference
    e = (d + 8) * 2.0 ** -24 * (30 * 0.6931471805599453 + 28)
    w = 2.0 ** -11 + 2 * e + 2 * n * 2.0 ** -24
    bound = (HALF[dtype] * ref + (1 + HALF[dtype]) * w * weighted + n * 2.0 ** -35 * float(v.float().max())
             + (2.0 ** -24 if dtype == FP16 else 0.0))
    err = (got.cpu().double() - ref).abs()
    assert (err <= bound).all(), (err / bound).max()
    assert (ref[..., 32:] > 4e-6).all()


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1, 2 ** 70])
def test_attention_windows_past_32_bits(window):
    """Longer than any table: no window, not what its low 32 bits say."""
    cache, table, start = _setup([90], [7], 1, 16, 64, seed=5)
    q = torch.randn(7, 2, 64, generator=_gen(4)).to(BF16).to(DEV)
    args = (q, _to(cache, DEV), _i32(table), _i32([90]), _i32(start))
    assert torch.equal(ops.kv_attention(*args, window=window), ops.kv_attention(*args))


def _poison_rest(cache, table, lens):
    """Everything of the cache that no request holds: NaN codes; scales of unused pages NaN."""
    page = cache.k.shape[2]
    k8, v8 = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    used = {}
    for b, n in enumerate(lens):
        for c in range(-(-n // page)):
            used[table[b][c]] = min(page, n - c * page)
    for p in range(cache.k.shape[0]):
        n = used.get(p, 0)
        k8[p, :, n:] = 0x7F
        v8[p, :, :, n:] = 0xFF
        if n == 0:
            cache.k_scale[p] = cache.v_scale[p] = float("nan")


def test_attention_ignores_what_no_request_holds():
    lens, rows = [1, 16, 30, 65, 200], [1, 3, 7, 2, 40]
    for d, page in ((128, 16), (64, 64)):
        cache, table, start = _setup(lens, rows, 2, page, d, seed=2, extra=5)
        q = torch.randn(start[-1], 4, d, generator=_gen(9)).to(BF16)
        clean = ops.kv_attention(q.to(DEV), _to(cache, DEV), _i32(table), _i32(lens), _i32(start))
        _poison_rest(cache, table, lens)
        got = ops.kv_attention(q.to(DEV), _to(cache, DEV), _i32(table), _i32(lens), _i32(start))
        assert torch.equal(clean, got)


def test_attention_pages_behind_the_window_may_be_gone():
    lens, rows, page, window = [300, 90], [4, 2], 16, 40
    cache, table, start = _setup(lens, rows, 2, page, 64, seed=5)
    q = torch.randn(6, 2, 64, generator=_gen(4)).to(BF16)
    args = (_i32(lens), _i32(start))
    want = ops.kv_attention(q.to(DEV), _to(cache, DEV), _i32(table), *args, window=window)
    for b, (n, r) in enumerate(zip(lens, rows)):
        for c in range((n - r - window + 1) // page):
            table[b][c] = (-1, 1 << 30, -(1 << 31))[c % 3]
    got = ops.kv_attention(q.to(DEV), _to(cache, DEV), _i32(table), *args, window=window)
    assert torch.equal(want, got)


def test_attention_missing_pages_and_poisoned_scales_give_nan():
    """Rows that see a token without a page, of a page with a NaN scale, or of a request longer than
    its table: NaN in every dimension.  Rows that do not, and other requests, are unharmed."""
    lens, rows, page, d = [100, 100, 100, 40], [60, 60, 60, 3], 16, 64
    cache, table, start = _setup(lens, rows, 2, page, d, seed=7)
    q = torch.randn(start[-1], 4, d, generator=_gen(4)).to(FP16).to(DEV)
    clean = ops.kv_attention(q, _to(cache, DEV), _i32(table), _i32(lens), _i32(start))
    table[0][4] = cache.k.shape[0]               # tokens 64..79
    cache.v_scale[table[1][5], 1] = float("nan")  # tokens 80..95 of kv head 1
    cache.k_scale[table[2][3], 0] = float("nan")  # tokens 48..63 of kv head 0
    dev = _to(cache, DEV)
    got = ops.kv_attention(q, dev, _i32(table), _i32(lens), _i32(start))
    want = torch.isnan(got)
    bad = torch.zeros_like(want)
    bad[64 - 40:60] = True
    bad[60 + 80 - 40:120, 2:] = True
    bad[120 + 48 - 40:180, :2] = True
    assert torch.equal(want, bad)
    assert torch.equal(got[~bad], clean[~bad])
    short = _i32(table)[:, :6]                   # 96 tokens: requests 0 to 2 do not fit
    got = ops.kv_attention(q, dev, short, _i32(lens), _i32(start))
    assert torch.isnan(got[:180]).all() and torch.equal(got[180:], clean[180:])
    got = ops.kv_attention(q, dev, _i32(table), _i32([2 ** 31 - 1] * 4), _i32(start))
    assert torch.isnan(got).all()
    # more rows than the table has room for, and a table without room
    for cols in (1, 0):
        got = ops.kv_attention(q, dev, _i32(table)[:, :cols], _i32(lens), _i32(start), window=7)
        assert torch.isnan(got).all()
    got = ops.kv_attention(q, dev, _i32(table)[:, :0], _i32([0, -3, 0, 0]), _i32(start))
    assert (got == 0).all()


@pytest.mark.parametrize("hq,d,page", [(4, 64, 16), (4, 256, 16), (4, 512, 64), (20, 128, 32)])
def test_attention_missing_pages_spare_earlier_rows_whatever_the_pool_holds(hq, d, page):
    """Rows in front of a missing page, in a tile with rows behind it, in a pool whose unheld places
    are NaN codes (a pool that was not zeroed)."""
    lens, rows = [200, 150], [90, 40]
    cache, table, start = _setup(lens, rows, 2, page, d, seed=3)
    free = [p for p in range(cache.k.shape[0]) if not any(p in r for r in table)]
    q = torch.randn(start[-1], hq, d, generator=_gen(4)).to(BF16).to(DEV)
    clean = ops.kv_attention(q, _to(cache, DEV), _i32(table), _i32(lens), _i32(start))
    _poison_rest(cache, table, lens)
    move = [free[0], *[p for p in range(cache.k.shape[0]) if p != free[0]]]  # page 0 is one that no request holds
    at = {old: new for new, old in enumerate(move)}
    cache = ops.KVCache(*[(x.view(torch.uint8)[move].view(x.dtype) if x.dtype == O.E4M3 else x[move]) for x in cache])
    cache.k_scale[0] = cache.v_scale[0] = 1.0
    table = [[at.get(p, -1) for p in r] for r in table]
    table[0][128 // page] = -1                 # tokens 128 to 128 + page
    table[1][128 // page] = cache.k.shape[0]
    got = ops.kv_attention(q, _to(cache, DEV), _i32(table), _i32(lens), _i32(start))
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[128 - 110:90] = True
    bad[90 + 128 - 110:] = True
    assert torch.equal(torch.isnan(got), bad)
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("window", [2 ** 31 - 1, 64, 63])
def test_attention_windows_around_the_table(window):
    """Windows as long as the table and longer, with rows that see nothing beside ones that do."""
    lens, rows, page = [40, 20, 48], [60, 3, 48], 16
    cache, table, start = _setup(lens, rows, 1, page, 64, seed=5)
    q = torch.randn(start[-1], 2, 64, generator=_gen(4)).to(BF16)
    got = ops.kv_attention(q.to(DEV), _to(cache, DEV), _i32(table), _i32(lens), _i32(start), window=window)
    ref, weighted, size = O.attention(q, cache, table, lens, start, 64 ** -0.5, window)
    _check_out(got, ref, weighted, size, 64, 48)


def test_attention_leaves_rows_behind_the_last_request():
    lens, rows = [20, 33], [2, 1]
    cache, table, start = _setup(lens, rows, 2, 16, 64, seed=1)
    q = torch.randn(7, 4, 64, generator=_gen(4)).to(BF16).to(DEV)
    q[3:] = float("nan")
    out = torch.full_like(q, 5.0)
    r = ops.kv_attention(q, _to(cache, DEV), _i32(table), _i32(lens), _i32(start), out=out)
    assert r is out and (out[3:] == 5).all() and torch.isfinite(out[:3]).all()
    # padded requests of a batch: no tokens, no rows
    pad = ops.kv_attention(q, _to(cache, DEV), _i32(table + [[-1] * len(table[0])] * 3), _i32(lens + [0, 0, 0]),
                           _i32(start + [3, 3, 3]))
    assert torch.equal(pad[:3], out[:3])
    # q_start that runs past the rows, or backwards: nothing outside them is touched
    for s in ([0, 2, 90], [0, 5, 2], [-4, 1, 3], [6, 7, 2 ** 31 - 1]):
        out.fill_(5.0)
        ops.kv_attention(q[:5], _to(cache, DEV), _i32(table), _i32(lens), _i32(s), out=out[:5])
        assert (out[5:] == 5).all()


def test_attention_strided_rows_and_outputs():
    lens = [50, 20, 64]
    cache, table, start = _setup(lens, [1] * 3, 2, 16, 128, seed=3)
    dev = _to(cache, DEV)
    wide = torch.randn(3, 8 * 128 + 8, generator=_gen(4)).to(BF16).to(DEV)
    q = wide[:, 4 * 128:8 * 128].unflatten(1, (4, 128))
    want = ops.kv_attention(q.contiguous(), dev, _i32(table), _i32(lens))
    assert torch.equal(want, ops.kv_attention(q, dev, _i32(table), _i32(lens)))
    odd = torch.empty(3 * 4 * 128 + 1, dtype=BF16, device=DEV)[1:].view(3, 4, 128)
    odd.copy_(q)
    assert torch.equal(want, ops.kv_attention(odd, dev, _i32(table), _i32(lens)))
    out = torch.zeros(4, 3, 136, dtype=BF16, device=DEV)
    view = out.transpose(0, 1)[..., :128]
    ops.kv_attention(q, dev, _i32(table), _i32(lens), out=view)
    assert torch.equal(view, want) and (out[..., 128:] == 0).all()
    big = torch.full((3, 90), -1, dtype=torch.int32, device=DEV)
    big[:, :len(table[0])] = _i32(table)
    assert torch.equal(want, ops.kv_attention(q, dev, big[:, :len(table[0])], _i32(lens)))


def test_cache_offsets_past_32_bits():
    """Pages more than 4 GiB into the pool, for the writer and the reader."""
    hk, page, d = 8, 256, 512
    pages = (5 << 30) // (hk * page * d)
    cache = ops.kv_cache(pages, hk, page, d, DEV)
    t = 300
    at = [pages - 1, 3]
    slots = torch.tensor([at[i // page] * page + i % page for i in range(t)], device=DEV)
    k = torch.randn(t, hk, d, generator=_gen(1)).to(BF16).to(DEV)
    v = torch.randn(t, hk, d, generator=_gen(2)).to(BF16).to(DEV)
    small = ops.kv_cache(2, hk, page, d, DEV)
    ops.kv_append(k, v, slots, cache)
    ops.kv_append(k, v, torch.arange(t, device=DEV), small)
    for x, y in zip(cache, small):
        x, y = (z.view(torch.uint8) if z.dtype == O.E4M3 else z for z in (x, y))
        assert torch.equal(x[at], y)
        assert not x[at[1] + 1:pages - 1].any()
    q = torch.randn(1, 16, d, generator=_gen(3)).to(BF16).to(DEV)
    a = ops.kv_attention(q, cache, _i32([at]), _i32([t]))
    assert torch.equal(a, ops.kv_attention(q, small, _i32([[0, 1]]), _i32([t])))


def test_attention_is_deterministic_and_runs_on_any_stream():
    lens = [3000, 40]
    cache, table, start = _setup(lens, [1, 1], 2, 16, 128, seed=11)
    dev = _to(cache, DEV)
    q = torch.randn(2, 8, 128, generator=_gen(4)).to(BF16).to(DEV)
    t, n = _i32(table), _i32(lens)
    want = ops.kv_attention(q, dev, t, n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:  # two calls under way at once, each with its own scratch
            with torch.cuda.stream(s):
                got.append(ops.kv_attention(q, dev, t, n))
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for x in got)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_steps_of_a_layer_in_two_graphs():
    """Slots, projections, rope, append and attention of a padded batch over steps, captured once
    for prompts and once for decoding (the two share the stream and the memory pool) and replayed
    with other lengths, against the same calls made eagerly and against the oracle."""
    hq, hk, d, page, h, b, cols = 4, 2, 64, 16, 128, 5, 12
    g = _gen(21)
    w = [tuple(x.to(DEV) for x in synth.linear_weights(h, n * d, 64, seed=n)) for n in (hq, hk, hk + 1)]
    w[2] = tuple(x[:, :hk * d].contiguous() for x in w[2])
    freq, _ = ops.rope_frequencies(d // 2, device=DEV)

    def step(st, rows):
        r = ops.kv_slots(st["ctx"], st["new"], st["table"], st["free"], st["used"], page, rows)
        q, k, v = (y.view(rows, -1, d) for y in ops.w4a16_linear_multi(st["x"][:rows], w, 64))
        q, k = ops.rope_rows(q, k, r.positions, freq, interleaved=True)
        ops.kv_append(k, v, r.slots, st["cache"])
        o = ops.kv_attention(q, st["cache"], st["table"], r.seq_lens, r.q_start, out=st["out"][:rows])
        st["ctx"].copy_(r.seq_lens)
        st["used"].copy_(r.status)
        return q, k, v, r, o

    def fresh():
        return {"ctx": _i32([0] * b), "new": _i32([0] * b), "free": torch.randperm(60, generator=_gen(1)).int().to(DEV),
                "table": torch.full((b, cols), -1, dtype=torch.int32, device=DEV), "used": _i32([0, 0, 0]),
                "cache": ops.kv_cache(60, hk, page, d, DEV), "x": torch.zeros(70, h, dtype=BF16, device=DEV),
                "out": torch.zeros(70, hq, d, dtype=BF16, device=DEV)}

    def reset(st, other):
        for n, x in st.items():
            for u, y in zip(x if n == "cache" else [x], other[n] if n == "cache" else [other[n]]):
                u.view(torch.uint8).copy_(y.view(torch.uint8))

    plan = [([33, 0, 17, 1, 9], 70), ([1, 0, 1, 1, 1], 8), ([1, 0, 1, 1, 1], 8), ([0, 40, 0, 2, 0], 70),
            ([1, 1, 1, 1, 0], 8), ([1, 1, 0, 1, 1], 8)]
    xs = [synth.activations(70, h, seed=i).to(DEV) for i in range(len(plan))]
    eager, replay = fresh(), fresh()
    graphs, side = {}, torch.cuda.Stream()
    with torch.cuda.stream(side):
        for rows in (70, 8):
            step(replay, rows)  # sets up what the linears keep between calls
    torch.cuda.synchronize()
    for rows in (70, 8):
        graphs[rows] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[rows], stream=side):
            step(replay, rows)
    reset(replay, eager)
    for i, (new, rows) in enumerate(plan):
        for st in (eager, replay):
            st["new"].copy_(_i32(new))
            st["x"].copy_(xs[i])
        before = _to(eager["cache"], "cpu")
        q, k, v, r, o = step(eager, rows)
        graphs[rows].replay()
        torch.cuda.synchronize()
        n = sum(new)
        for name in ("ctx", "table", "used"):
            assert torch.equal(eager[name], replay[name]), (i, name)
        _same_cache(replay["cache"], _to(eager["cache"], "cpu"))
        assert torch.equal(eager["out"][:n], replay["out"][:n]), i
        want = O.append(k.cpu(), v.cpu(), r.slots.tolist(), before)
        _same_cache(eager["cache"], want)
        ref, weighted, size = O.attention(q.cpu()[:n], want, eager["table"].tolist(), r.seq_lens.tolist(),
                                          r.q_start.tolist(), d ** -0.5)
        _check_out(o[:n], ref, weighted, size, d, 64)


def test_rollbacks_over_page_ends_lose_no_page():
    """Verify steps whose drafts are rejected in part, in one graph: the pages that a request no
    longer reaches go back on the list on the device, and no page is lost or held twice."""
    b, page, cols, draft, total = 6, 16, 40, 7, 200
    st = {"ctx": _i32([3, 15, 16, 31, 40, 250]), "new": _i32([draft] * b), "keep": _i32([0] * b)}
    store = torch.cat([torch.randperm(total, generator=_gen(1)).int(), torch.tensor([-1], dtype=torch.int32)]).to(DEV)
    table, used = torch.full((b, cols), -1, dtype=torch.int32, device=DEV), _i32([0, 0, 0])

    def give_back(had, keep, table, store, used, page):
        first = (keep + page - 1) // page
        gone = first < (had + page - 1) // page
        at = first.clamp(max=table.shape[1] - 1).long()[:, None]
        pages = table.gather(1, at)[:, 0]
        gone &= pages >= 0
        place = torch.where(gone, used[0] - gone.cumsum(0), store.numel() - 1)
        store.scatter_(0, place, pages)
        used[0] -= gone.sum()

    def step():
        r = ops.kv_slots(st["ctx"], st["new"], table, store[:-1], used, page, b * draft)
        used.copy_(r.status)
        st["ctx"].add_(st["keep"])  # of the draft, `keep` tokens are right
        give_back(r.seq_lens, st["ctx"], table, store, used, page)
        return r

    zero = torch.zeros_like(st["ctx"])
    r = ops.kv_slots(zero, st["ctx"], table, store[:-1], used, page, int(st["ctx"].sum()))
    used.copy_(r.status)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()  # keeps nothing: what it took goes back
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step()
    rng = random.Random(2)
    lens = st["ctx"].tolist()
    for _ in range(40):
        keep = [rng.randint(0, draft) for _ in range(b)]
        st["keep"].copy_(_i32(keep))
        graph.replay()
        torch.cuda.synchronize()
        lens = [n + k for n, k in zip(lens, keep)]
        assert st["ctx"].tolist() == lens
        n, rows = int(used[0]), table.tolist()
        held = [p for row, ln in zip(rows, lens) for p in row[:-(-ln // page)]]
        assert n == len(held) == sum(-(-ln // page) for ln in lens) and used.tolist()[1:] == [0, 0]
        assert sorted(held + store[n:-1].tolist()) == list(range(total))


# ---------------------------------------------------------------------------
# refusals of the torch-facing calls
# ---------------------------------------------------------------------------
def test_results_that_share_elements_are_refused():
    """Rows or heads of a result on the same memory would be written by several workgroups at once."""
    cache = ops.kv_cache(4, 2, 16, 64, DEV)
    q = torch.zeros(3, 4, 64, dtype=BF16, device=DEV)
    t, n, s = _i32([[0, 1]] * 3), _i32([1, 2, 3]), torch.zeros(3, dtype=torch.int64, device=DEV)
    freq = ops.rope_frequencies(64, device=DEV)[0]
    for out in (torch.zeros_like(q[:1]).expand(3, 4, 64), torch.zeros_like(q[:, :1]).expand(3, 4, 64)):
        with pytest.raises(ValueError, match="broadcast"):
            ops.kv_attention(q, cache, t, n, out=out)
    one = torch.zeros(3, 4, 64, dtype=BF16, device=DEV).transpose(0, 1)[:, :1].transpose(0, 1)  # a single row of any stride
    assert ops.kv_attention(q[:1], cache, t[:1], n[:1], out=one) is one
    for k in (q, q[:, :2]):
        with pytest.raises(ValueError, match="same elements"):
            ops.rope_rows(q, k, s, freq, inplace=True)
        ops.rope_rows(q, k, s, freq)
    ops.rope_rows(q[:, :3], q[:, 3:], s, freq, inplace=True)


def test_counts_past_31_bits_are_refused():
    """Not served as what their low 32 bits say."""
    n = 2 ** 32 + 3
    cache = ops.kv_cache(4, 2, 16, 64, DEV)
    row = torch.zeros(1, 2, 64, dtype=BF16, device=DEV)
    slots = torch.empty(n, dtype=torch.int64, device=DEV)
    ints = slots.view(torch.int32)[:n]
    one, table = _i32([1]), _i32([[0, 1]])
    freq = ops.rope_frequencies(64, device=DEV)[0]
    calls = [
        lambda: ops.kv_append(row.expand(n, 2, 64), row.expand(n, 2, 64), slots, cache),
        lambda: ops.rope_rows(row.expand(n, 2, 64), None, slots, freq),
        lambda: ops.kv_slots(one, one, table, ints, one, 16, 3),
        lambda: ops.kv_slots(one, one, ints[None], one, one, 16, 3),
        lambda: ops.kv_slots(ints, ints, table.expand(n, 2), one, one, 16, 3),
        lambda: ops.kv_attention(row.expand(n, 2, 64), cache, table, one, _i32([0, 1])),
        lambda: ops.kv_attention(row, cache, ints[None], one),
        lambda: ops.kv_attention(row.expand(n, 2, 64), cache, table.expand(n, 2), ints),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
            print("no refusal of call", i)


def test_refusals():
    cache = ops.kv_cache(4, 2, 16, 64, DEV)
    x = torch.zeros(3, 2, 64, dtype=BF16, device=DEV)
    s = torch.zeros(3, dtype=torch.int64, device=DEV)
    q = torch.zeros(3, 4, 64, dtype=BF16, device=DEV)
    t, n = _i32([[0, 1]] * 3), _i32([1, 2, 3])
    for kw in (dict(page_size=24), dict(head_dim=96), dict(num_pages=0)):
        with pytest.raises(ValueError):
            ops.kv_cache(**{**dict(num_pages=4, kv_heads=2, page_size=16, head_dim=64, device=DEV), **kw})
    bad = [
        (ValueError, lambda: ops.kv_append(x[:, :1], x[:, :1], s, cache)),
        (ValueError, lambda: ops.kv_append(x, x[:2], s, cache)),
        (ValueError, lambda: ops.kv_append(x, x, s[:2], cache)),
        (TypeError, lambda: ops.kv_append(x, x, s.int(), cache)),
        (TypeError, lambda: ops.kv_append(x, x.float(), s, cache)),
        (TypeError, lambda: ops.kv_append(x.cpu(), x, s, cache)),
        (ValueError, lambda: ops.kv_append(x.transpose(1, 2).contiguous().transpose(1, 2), x, s, cache)),
        (ValueError, lambda: ops.kv_append(x, x, s, cache._replace(v=cache.k))),
        (TypeError, lambda: ops.kv_append(x, x, s, cache._replace(k=cache.k.view(torch.uint8)))),
        (ValueError, lambda: ops.kv_append(x, x, s, cache._replace(k_scale=cache.k_scale[:3]))),
        (TypeError, lambda: ops.kv_attention(q.float(), cache, t, n)),
        (ValueError, lambda: ops.kv_attention(q[:, :3], cache, t, n)),
        (ValueError, lambda: ops.kv_attention(q, cache, t[:2], n)),
        (ValueError, lambda: ops.kv_attention(q[:2], cache, t, n)),
        (ValueError, lambda: ops.kv_attention(q, cache, t, n, _i32([0, 3]))),
        (TypeError, lambda: ops.kv_attention(q, cache, t, n.long())),
        (TypeError, lambda: ops.kv_attention(q, cache, t.long(), n)),
        (ValueError, lambda: ops.kv_attention(q, cache, t, n, window=-1)),
        (ValueError, lambda: ops.kv_attention(q, cache, t, n, out=q)),
        (ValueError, lambda: ops.kv_attention(q, cache, t, n, out=torch.zeros(3, 4, 65, dtype=BF16, device=DEV)[..., :64])),
        (ValueError, lambda: ops.kv_attention(q, cache, t[:1].expand(3, 2), n)),
        (TypeError, lambda: ops.rope_rows(q, x, s.int(), ops.rope_frequencies(64, device=DEV)[0])),
        (TypeError, lambda: ops.rope_rows(q, x, s, ops.rope_frequencies(64, device=DEV)[0].float())),
        (ValueError, lambda: ops.rope_rows(q, x, s, ops.rope_frequencies(66, device=DEV)[0])),
        (ValueError, lambda: ops.rope_rows(q, x[:2], s, ops.rope_frequencies(64, device=DEV)[0])),
        (ValueError, lambda: ops.rope_rows(q[:, :1].expand(3, 4, 64), None, s, ops.rope_frequencies(64, device=DEV)[0],
                                           inplace=True)),
        (ValueError, lambda: ops.rope_frequencies(7)),
        (ValueError, lambda: ops.rope_frequencies(8, scaling="other")),
        (ValueError, lambda: ops.kv_slots(n, n[:2], t, n, n, 16, 5)),
        (ValueError, lambda: ops.kv_slots(n, n, t, n, n, 20, 5)),
        (TypeError, lambda: ops.kv_slots(n.long(), n, t, n, n, 16, 5)),
        (ValueError, lambda: ops.kv_slots(n, n, t, n, n, 16, -1)),
        (L.GIError, lambda: ops.kv_slots(_i32([0] * 9000), _i32([0] * 9000), _i32([[0]] * 9000), n, n, 16, 5)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            print("no refusal of call", i)
