"""Host-side argument checks of the paged-cache entry points (they return before any HIP call),
and the oracle's own rounding."""
import ctypes
import math

import pytest
import torch

from gemmainfer_amd import _lib as L
from gemmainfer_amd import ops
from oracle import kv_oracle as O

VP = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(8)


@pytest.fixture(scope="module")
def lib():
    if not L.LIB_PATH.exists():
        from gemmainfer_amd import build
        build.build(verbose=False)
    return L.load()


def _call(lib, fn, args, over):
    a = {**args, **over}
    return getattr(lib, fn)(*a.values()), lib.gi_last_error().decode()


ROPE = dict(q=VP, qo=VP, k=VP, ko=VP, pos=VP, freq=VP, dtype=L.DTYPE_BF16, T=2, Hq=4, Hk=2, D=64, rot=64, inter=0,
            mscale=1.0, a=256, b=64, c=256, d=64, e=128, f=64, g=128, h=64, stream=None)


@pytest.mark.parametrize("over,code,frag", [
    (dict(dtype=L.DTYPE_INT32), L.GI_ERR_UNSUPPORTED, "bf16, fp16 or fp32"),
    (dict(rot=63), L.GI_ERR_INVALID_ARG, "rotary_dim"),
    (dict(rot=66), L.GI_ERR_INVALID_ARG, "rotary_dim"),
    (dict(rot=0), L.GI_ERR_INVALID_ARG, "rotary_dim"),
    (dict(D=2048, rot=1026), L.GI_ERR_UNSUPPORTED, "1024"),
    (dict(T=-1), L.GI_ERR_INVALID_ARG, "T"),
    (dict(pos=None), L.GI_ERR_INVALID_ARG, "null"),
    (dict(ko=None), L.GI_ERR_INVALID_ARG, "null"),
])
def test_rope_rows_refuses(lib, over, code, frag):
    st, msg = _call(lib, "gi_rope_rows", ROPE, over)
    assert st == code and frag in msg


SLOTS = dict(ctx=VP, new=VP, B=2, table=VP, cols=4, stride=4, free=VP, n_free=3, used=VP, page=16, slots=VP, pos=VP,
             n=5, start=VP, lens=VP, status=VP, stream=None)


@pytest.mark.parametrize("over,code,frag", [
    (dict(page=24), L.GI_ERR_INVALID_ARG, "page_size"),
    (dict(page=8), L.GI_ERR_INVALID_ARG, "page_size"),
    (dict(B=8193), L.GI_ERR_UNSUPPORTED, "8192"),
    (dict(B=-1), L.GI_ERR_INVALID_ARG, "negative"),
    (dict(stride=3), L.GI_ERR_INVALID_ARG, "table_stride"),
    (dict(table=None), L.GI_ERR_INVALID_ARG, "null"),
    (dict(used=None), L.GI_ERR_INVALID_ARG, "null"),
    (dict(slots=None), L.GI_ERR_INVALID_ARG, "null"),
])
def test_kv_slots_refuses(lib, over, code, frag):
    st, msg = _call(lib, "gi_kv_slots", SLOTS, over)
    assert st == code and frag in msg


APPEND = dict(k=VP, v=VP, dtype=L.DTYPE_BF16, a=128, b=64, c=128, d=64, slots=VP, T=2, Hk=2, D=64, page=16, pages=4,
              kc=VP, vc=VP, ks=VP, vs=VP, stream=None)


@pytest.mark.parametrize("over,code,frag", [
    (dict(dtype=L.DTYPE_INT64), L.GI_ERR_UNSUPPORTED, "bf16, fp16 or fp32"),
    (dict(page=17), L.GI_ERR_INVALID_ARG, "page_size"),
    (dict(D=60), L.GI_ERR_INVALID_ARG, "multiple of 8"),
    (dict(D=2048), L.GI_ERR_INVALID_ARG, "1024"),
    (dict(Hk=70000), L.GI_ERR_UNSUPPORTED, "65535"),
    (dict(slots=None), L.GI_ERR_INVALID_ARG, "null"),
    (dict(kc=ODD), L.GI_ERR_INVALID_ARG, "aligned"),
    (dict(T=0, k=None), L.GI_OK, ""),
    (dict(pages=0, kc=None), L.GI_OK, ""),
])
def test_kv_append_refuses(lib, over, code, frag):
    st, msg = _call(lib, "gi_kv_append", APPEND, over)
    assert st == code and (code == L.GI_OK or frag in msg)


ATTN = dict(q=VP, dtype=L.DTYPE_BF16, a=256, b=64, kc=VP, vc=VP, ks=VP, vs=VP, table=VP, cols=4, stride=4, lens=VP,
            start=VP, out=VP, c=256, d=64, T=3, B=2, Hq=4, Hk=2, D=64, page=16, pages=4, scale=0.125, window=0, ws=None,
            wsb=0, stream=None)


@pytest.mark.parametrize("over,code,frag", [
    (dict(), L.GI_ERR_WORKSPACE, "workspace"),
    (dict(cols=400, stride=400, ws=VP, wsb=1024), L.GI_ERR_WORKSPACE, "workspace"),
    (dict(dtype=L.DTYPE_FP32), L.GI_ERR_UNSUPPORTED, "bf16 or fp16"),
    (dict(Hq=5), L.GI_ERR_INVALID_ARG, "multiple of Hk"),
    (dict(D=96), L.GI_ERR_UNSUPPORTED, "64, 128, 256 and 512"),
    (dict(page=48), L.GI_ERR_INVALID_ARG, "page_size"),
    (dict(start=None), L.GI_ERR_INVALID_ARG, "one row a request"),
    (dict(scale=float("nan")), L.GI_ERR_INVALID_ARG, "scale"),
    (dict(window=-1), L.GI_ERR_INVALID_ARG, "window"),
    (dict(pages=0), L.GI_ERR_INVALID_ARG, "no pages"),
    (dict(lens=None), L.GI_ERR_INVALID_ARG, "null"),
    (dict(q=ODD), L.GI_ERR_INVALID_ARG, "aligned"),
    (dict(a=260), L.GI_ERR_INVALID_ARG, "strides"),
    (dict(stride=3), L.GI_ERR_INVALID_ARG, "table_stride"),
    (dict(cols=1 << 27, stride=1 << 27), L.GI_ERR_UNSUPPORTED, "2^30"),
    (dict(T=0, q=None), L.GI_OK, ""),
])
def test_kv_attention_refuses(lib, over, code, frag):
    st, msg = _call(lib, "gi_kv_attention", ATTN, over)
    assert st == code and (code == L.GI_OK or frag in msg)


def test_largest_counts_are_refused(lib):
    """Where the kernels' own counting would end: refused before any pointer is looked at."""
    st, msg = _call(lib, "gi_kv_append", APPEND, dict(T=(1 << 30) + 1, k=None))
    assert st == L.GI_ERR_UNSUPPORTED and "2^30" in msg
    st, msg = _call(lib, "gi_kv_attention", ATTN, dict(B=(1 << 20) + 1, q=None))
    assert st == L.GI_ERR_UNSUPPORTED and "2^20" in msg
    st, msg = _call(lib, "gi_kv_attention", ATTN, dict(B=1 << 20, T=1 << 20, start=None))
    assert st == L.GI_ERR_WORKSPACE


def test_more_heads_than_a_grid_is_wide_are_refused(lib):
    heads = (1 << 23) + 1
    st, msg = _call(lib, "gi_kv_attention", ATTN, dict(Hq=heads, Hk=heads, q=None))
    assert st == L.GI_ERR_UNSUPPORTED and "2^23" in msg
    assert lib.gi_kv_attention_workspace_bytes(3, 2, heads, heads, 64, 64) == 0
    st, msg = _call(lib, "gi_kv_attention", ATTN, dict(Hq=1 << 23, Hk=1 << 23))
    assert st == L.GI_ERR_WORKSPACE


def test_workspace_query_is_host_only(lib):
    q = lib.gi_kv_attention_workspace_bytes
    for bad in ((0, 1, 16, 8, 256), (1, 0, 16, 8, 256), (1, 1, 15, 8, 256), (1, 1, 16, 8, 96)):
        assert q(*bad, 4096) == 0
    assert 0 < q(1, 1, 16, 8, 256, 256) <= 64         # one chunk: nothing to join
    assert q(1, 1, 16, 8, 256, 4096) < 1 << 24
    assert q(64, 64, 16, 8, 256, 1 << 20) < 1 << 27    # bounded by what the chip holds, not by the lengths


@pytest.mark.parametrize("hq,hk,d", [(16, 8, 256), (16, 2, 512), (32, 8, 128), (12, 4, 64), (40, 1, 64), (64, 64, 64)])
def test_workspace_query_does_not_shrink(lib, hq, hk, d):
    """One workspace for the largest T, B and table serves every smaller call."""
    q = lib.gi_kv_attention_workspace_bytes
    sizes = [1, 2, 3, 7, 16, 17, 33, 64, 65, 100, 512, 4000]
    for tokens in (256, 272, 4096, 1 << 17):
        need = {(t, b): q(t, b, hq, hk, d, tokens) for t in sizes for b in sizes}
        for (t, b), n in need.items():
            assert n >= max(need[x, y] for x in sizes if x <= t for y in sizes if y <= b), (t, b, tokens)
            assert n <= q(t, b, hq, hk, d, 2 * tokens)


def test_device_calls_reject_host_tensors():
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(TypeError, match="device tensors"):
        ops.rope_rows(x, None, i, torch.zeros(32, dtype=torch.float64))
    with pytest.raises(TypeError, match="device tensors"):
        ops.kv_append(x, x, i, ops.kv_cache(1, 1, 16, 64, "cpu"))


@pytest.mark.parametrize("rotary,base,factor,original,fast,slow", [
    (128, 1e4, 16.0, 8192, 32.0, 1.0), (64, 5e5, 4.0, 4096, 32.0, 1.0), (256, 1e6, 40.0, 32768, 64.0, 2.0),
    (16, 1e4, 2.0, 100, 3.0, 0.5)])
def test_yarn_ramp_is_linear_in_the_turns(rotary, base, factor, original, fast, slow):
    """Every frequency, one at a time: kept over `fast` turns in `original` tokens, divided by `factor` under
    `slow`, and between them the share (turns - slow) / (fast - slow) of it is kept."""
    got, mscale = ops.rope_frequencies(rotary, base, scaling="yarn", factor=factor, original_len=original, fast=fast,
                                       slow=slow, device="cpu")
    seen = set()
    for i in range(rotary // 2):
        f = base ** (-2.0 * i / rotary)
        turns = original * f / (2 * math.pi)
        keep = 1.0 if turns >= fast else 0.0 if turns <= slow else (turns - slow) / (fast - slow)
        seen.add(0 if turns <= slow else 2 if turns >= fast else 1)
        assert abs(float(got[i]) - (keep * f + (1 - keep) * f / factor)) <= 1e-13 * f
    assert seen == {0, 1, 2} and abs(mscale - (0.1 * math.log(factor) + 1)) < 1e-15


def test_oracle_rounds_like_torch():
    x = torch.cat([torch.randn(20000, generator=torch.Generator().manual_seed(0)) * 40,
                   torch.arange(-448, 449) / 64.0, torch.arange(-64, 65) / 2048.0]).clamp(-448, 448)
    assert torch.equal(O.to_e4m3(x.double()), x.to(O.E4M3).double())
    assert O.page_scale(448.0) == 1.0 and O.page_scale(448.5) == 2.0 and O.page_scale(0.0) == 2.0 ** -40
    assert O.page_scale(448.0 * 2 ** 40) == 2.0 ** 40 and O.page_scale(float("inf")) != O.page_scale(float("inf"))


def test_oracle_slots_by_hand():
    s, pos, start, lens, status, table = O.slots([3, 0], [14, 2], [[7, -1], [-1, -1]], [4, 9, 5], 1, 16, 18)
    assert s[:13] == [7 * 16 + 3 + i for i in range(13)] and s[13] == 9 * 16 and s[14:] == [80, 81, -1, -1]
    assert pos == [*range(3, 17), 0, 1, 0, 0] and start == [0, 14, 16] and lens == [17, 2]
    assert status == [3, 0, 0] and table == [[7, 9], [5, -1]]
