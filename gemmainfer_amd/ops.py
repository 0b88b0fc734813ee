"""torch-facing wrappers over the C ABI (device tensors only).

Every function here takes tensors on a ROCm device, checks shapes/dtypes the
way the reference's call sites imply, passes raw pointers plus torch's current
HIP stream to libgemmainfer_amd.so, and never synchronises.  Scratch
("workspace") memory is allocated once per (device, stream) through torch's
caching allocator, zero-filled once, and reused: the kernels leave it zeroed.

Reference entry points mirrored (GemmaInfer paths):
  fused_batched_moe   csrc/pybind.cpp:247-271 -> csrc/marlin.cu:612-702
  marlin_w4a16        csrc/pybind.cpp:182-196 -> csrc/marlin.cu:704-856
  route_topk_softmax  gemmainfer/models/gemma.py:77-80
  softcapping         csrc/pybind.cpp:169-180 -> csrc/softcapping.cu:21-47
  rmsnorm             csrc/pybind.cpp:137-151 -> csrc/rmsnorm.cu:75-114
  fused_rope_inplace  csrc/pybind.cpp:153-167 -> csrc/rmsnorm.cu:166-231

Without a native counterpart there (torch statements of
gemmainfer/kernels/attention.py:135-277): attention over an 8-bit paged K/V
cache -- kv_cache, kv_slots, rope_frequencies, rope_rows, kv_append,
kv_attention.
"""
from __future__ import annotations

import ctypes
import math
import threading
from typing import NamedTuple, Optional

import torch

from . import _lib as L

_DTYPE_CODE = {
    torch.bfloat16: L.DTYPE_BF16,
    torch.float16: L.DTYPE_FP16,
    torch.float32: L.DTYPE_FP32,
    torch.int32: L.DTYPE_INT32,
    torch.int64: L.DTYPE_INT64,
}


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


# The handle of torch's current stream without building a Stream object (2 us of each call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: torch.device) -> ctypes.c_void_p:
    if _raw_stream is not None and device.index is not None:
        return ctypes.c_void_p(_raw_stream(device.index))
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _require(cond: bool, msg: str, exc=ValueError) -> None:
    if not cond:
        raise exc(msg)


def _on_device(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if t.device != dev or not t.is_cuda:
            if not all(u.is_cuda for u in tensors):
                raise TypeError("gemmainfer_amd ops take ROCm device tensors only")
            raise ValueError(f"all tensors must be on {dev}, got {t.device}")
    return dev


# ---------------------------------------------------------------------------
# workspaces
# ---------------------------------------------------------------------------
class _WorkspacePool:
    """One zero-filled uint8 buffer per (kind, device, stream), grown on demand."""

    def __init__(self):
        self._bufs: dict[tuple, torch.Tensor] = {}
        self._lock = threading.Lock()

    def get(self, kind: str, device: torch.device, nbytes: int) -> torch.Tensor:
        stream = torch.cuda.current_stream(device).cuda_stream
        key = (kind, device.index, stream)
        with self._lock:
            buf = self._bufs.get(key)
            if buf is None or buf.numel() < nbytes:
                size = max(nbytes, 1 << 16)
                size = (size + 4095) // 4096 * 4096
                buf = torch.zeros(size, dtype=torch.uint8, device=device)
                self._bufs[key] = buf
            return buf

    def all(self, kind: str, device: torch.device):
        with self._lock:
            return [b for (k, d, _), b in self._bufs.items() if k == kind and d == device.index]


_WS = _WorkspacePool()


def _device_index(device) -> int:
    if device is None:
        return torch.cuda.current_device()
    d = torch.device(device)
    return torch.cuda.current_device() if d.index is None else d.index


def workspace_status(device=None) -> int:
    """OR of the device status words of every MoE workspace on ``device`` and
    of the device's host-visible error flag, clearing them (synchronises).
    0 means no kernel reported an error (``gemmainfer_amd._lib.DEVICE_SPIN_TIMEOUT``
    = a bounded wait gave up)."""
    device = torch.device("cuda", _device_index(device))
    lib = L.load()
    out = 0
    for buf in _WS.all("moe", device):
        st = ctypes.c_int32(0)
        L.check(lib.gi_workspace_status(_ptr(buf), buf.numel(), ctypes.byref(st), _stream(device)),
                "workspace_status")
        out |= st.value
    flags = lib.gi_device_error_flags(device.index, 1)
    return out | max(flags, 0)


def raise_pending_device_error(device=None) -> None:
    """Raise GIError(GI_ERR_DEVICE) if a kernel on ``device`` reported an error
    since the last check.  Reads a host-memory flag the kernels write: no
    synchronisation.  The MoE entry points call it before launching, so a
    failure surfaces at the next call (the failed call's outputs that could
    not be completed hold NaN).  The device's MoE workspaces are re-zeroed."""
    idx = _device_index(device)
    flags = L.load().gi_device_error_flags(idx, 1)
    if flags > 0:
        for buf in _WS.all("moe", torch.device("cuda", idx)):
            buf.zero_()
        raise L.GIError(L.GI_ERR_DEVICE,
                        f"a MoE kernel on cuda:{idx} reported device error bits {flags:#x} "
                        "(a bounded wait gave up; the outputs it could not complete hold NaN)")


# ---------------------------------------------------------------------------
# MoE
# ---------------------------------------------------------------------------
def _moe_weight_shapes(x, gu_packed, gu_scales, d_packed, d_scales):
    _require(x.dim() == 2, f"x must be [M, H], got {tuple(x.shape)}")
    m, h = x.shape
    _require(gu_packed.dim() == 3 and gu_packed.dtype == torch.int32,
             "gate_up_packed must be int32 [E, H/8, 2I]")
    e, hp, two_i = gu_packed.shape
    _require(hp * 8 == h, f"gate_up_packed.shape[1]*8 ({hp * 8}) must equal H ({h})")
    _require(two_i % 2 == 0, "gate_up_packed last dim must be 2*I")
    i = two_i // 2
    _require(gu_scales.dim() == 3 and gu_scales.shape[0] == e and gu_scales.shape[2] == two_i,
             f"gate_up_scales must be [E, groups, 2I], got {tuple(gu_scales.shape)}")
    _require(d_packed.dim() == 3 and d_packed.dtype == torch.int32 and
             tuple(d_packed.shape) == (e, i // 8, h),
             f"down_packed must be int32 [E, I/8, H] = {(e, i // 8, h)}, got {tuple(d_packed.shape)}")
    _require(d_scales.dim() == 3 and d_scales.shape[0] == e and d_scales.shape[2] == h,
             f"down_scales must be [E, groups, H], got {tuple(d_scales.shape)}")
    for name, t in (("gate_up_scales", gu_scales), ("down_scales", d_scales)):
        _require(t.dtype == x.dtype, f"{name} dtype {t.dtype} must match x dtype {x.dtype}", TypeError)
    for name, t in (("gate_up_packed", gu_packed), ("gate_up_scales", gu_scales),
                    ("down_packed", d_packed), ("down_scales", d_scales)):
        _require(t.is_contiguous(), f"{name} must be contiguous")
    return m, h, i, e


def _require_bf16(x: torch.Tensor, who: str) -> None:
    if x.dtype != torch.bfloat16:
        raise NotImplementedError(
            f"{who}: the gfx950 kernels implement bf16 activations; got {x.dtype}")


_ACT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _require_act_dtype(x: torch.Tensor, who: str) -> None:
    """bf16, fp16 or fp32 activations (the reference's dispatch, marlin.cu:694-700,
    :764-842).  bf16 runs the tuned kernels; so do fp16 MoE calls (caller-given
    ids) and fp16 linears of more than 16 rows; the rest run VALU kernels."""
    if x.dtype not in _ACT_DTYPES:
        raise TypeError(f"{who}: activations must be bf16, fp16 or fp32; got {x.dtype}")


def fused_batched_moe(x, gate_up_packed, gate_up_scales, down_packed, down_scales,
                      expert_indices, expert_weights, out, group_size, *, spin_limit: int = 0):
    """out += sum over slots of w * expert(x)  (drop-in for gemmainfer_csrc.fused_batched_moe).

    Semantics of the reference (csrc/marlin.cu:612-702): M = x.size(0),
    top_k = numel(expert_indices) / M, ids outside [0, E) are skipped, the
    weights are cast to x's dtype, and the result is ADDED to ``out`` (the
    caller zeroes it, gemma.py:82).  Unlike the reference there is no cap on
    how many slots share an expert (marlin.cu:325) and no 128-slot limit
    (:300); the combine is a fixed-order fp32 sum with one rounding to x's
    dtype.  x, the scales and out are bf16, fp16 or fp32 (all the same).
    """
    dev = _on_device(x, gate_up_packed, gate_up_scales, down_packed, down_scales,
                     expert_indices, expert_weights, out)
    raise_pending_device_error(dev)
    _require_act_dtype(x, "fused_batched_moe")
    m, h, i, e = _moe_weight_shapes(x, gate_up_packed, gate_up_scales, down_packed, down_scales)
    _require(isinstance(group_size, int) and group_size > 0 and group_size % 8 == 0,
             f"group_size must be a positive multiple of 8, got {group_size}")
    _require(tuple(out.shape) == (m, h), f"out must be [M, H] = {(m, h)}, got {tuple(out.shape)}")
    _require(out.dtype == x.dtype, "out dtype must match x", TypeError)
    if m == 0:
        return
    n_slots = expert_indices.numel()
    _require(n_slots % m == 0 and n_slots > 0,
             f"numel(expert_indices) ({n_slots}) must be a positive multiple of M ({m})")
    top_k = n_slots // m
    _require(expert_weights.numel() == n_slots,
             f"expert_weights has {expert_weights.numel()} elements, expected {n_slots}")
    idx = expert_indices
    if idx.dtype not in (torch.int32, torch.int64):
        idx = idx.to(torch.int32)
    idx = idx.contiguous()
    w = expert_weights
    if w.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        w = w.to(torch.float32)
    w = w.contiguous()
    xc = x.contiguous()
    oc = out if out.is_contiguous() else out.contiguous()
    lib = L.load()
    nbytes = lib.gi_fused_moe_workspace_bytes(m, top_k, h, i, e)
    ws = _WS.get("moe", dev, nbytes)
    L.check(lib.gi_fused_batched_moe(
        _ptr(xc), _DTYPE_CODE[x.dtype], _ptr(gate_up_packed), _ptr(gate_up_scales),
        gate_up_scales.shape[1], _ptr(down_packed), _ptr(down_scales), down_scales.shape[1],
        _ptr(idx), _DTYPE_CODE[idx.dtype], _ptr(w), _DTYPE_CODE[w.dtype], _ptr(oc),
        m, h, i, e, top_k, int(group_size), _ptr(ws), ws.numel(), int(spin_limit),
        _stream(dev)), "fused_batched_moe")
    if oc is not out:
        out.copy_(oc)


def moe_layer(x, router_logits, gate_up_packed, gate_up_scales, down_packed, down_scales,
              top_k, group_size, expert_scale=None, out=None, *, spin_limit: int = 0):
    """Router tail + fused MoE (gemma.py:77-98): one launch per 8 rows up to
    11 rows (up to 24 at decode widths with few experts or a small top_k), and
    from there the grouped-GEMM prefill path (routing with the align, gate/up,
    down and combine launches).

    Returns (out [M, H] bf16 -- overwritten, idx int32 [M, top_k],
    weights bf16 [M, top_k]).
    """
    dev = _on_device(x, router_logits, gate_up_packed, gate_up_scales, down_packed, down_scales)
    raise_pending_device_error(dev)
    _require_bf16(x, "moe_layer")
    m, h, i, e = _moe_weight_shapes(x, gate_up_packed, gate_up_scales, down_packed, down_scales)
    _require(router_logits.dim() == 2 and tuple(router_logits.shape) == (m, e),
             f"router_logits must be [M, E] = {(m, e)}, got {tuple(router_logits.shape)}")
    _require(router_logits.dtype in (torch.bfloat16, torch.float32),
             "router_logits must be bf16 or fp32", TypeError)
    _require(0 < top_k <= min(e, 64), f"top_k must be in [1, min(E, 64)], got {top_k}")
    if expert_scale is not None:
        _on_device(x, expert_scale)
        _require(expert_scale.numel() == e, "expert_scale must have E elements")
        expert_scale = expert_scale.to(torch.float32).contiguous()
    if out is None:
        out = torch.empty_like(x)
    _require(tuple(out.shape) == (m, h) and out.dtype == x.dtype and out.is_contiguous(),
             "out must be a contiguous bf16 [M, H] tensor")
    idx = torch.empty((m, top_k), dtype=torch.int32, device=dev)
    w = torch.empty((m, top_k), dtype=torch.bfloat16, device=dev)
    if m == 0:
        return out, idx, w
    logits = router_logits.contiguous()
    lib = L.load()
    nbytes = lib.gi_fused_moe_workspace_bytes(m, top_k, h, i, e)
    ws = _WS.get("moe", dev, nbytes)
    L.check(lib.gi_moe_layer_from_logits(
        _ptr(x.contiguous()), L.DTYPE_BF16, _ptr(logits), _DTYPE_CODE[logits.dtype],
        _ptr(expert_scale), _ptr(gate_up_packed), _ptr(gate_up_scales), gate_up_scales.shape[1],
        _ptr(down_packed), _ptr(down_scales), down_scales.shape[1], _ptr(out), _ptr(idx),
        _ptr(w), m, h, i, e, int(top_k), int(group_size), _ptr(ws), ws.numel(),
        int(spin_limit), _stream(dev)), "moe_layer")
    return out, idx, w


def _router_inputs(x, router_scale, gate_weight, who):
    dev = _on_device(x, gate_weight)
    _require_bf16(x, who)
    _require(x.dim() == 2, f"{who}: x must be [M, H]")
    m, h = x.shape
    _require(gate_weight.dim() == 2 and gate_weight.shape[1] == h,
             f"{who}: gate weight must be [E, H={h}], got {tuple(gate_weight.shape)}")
    _require(gate_weight.dtype == torch.bfloat16, f"{who}: gate weight must be bf16", TypeError)
    if router_scale is not None:
        _on_device(x, router_scale)
        _require(router_scale.numel() == h and router_scale.dtype == torch.bfloat16,
                 f"{who}: router_scale must be a bf16 tensor of H={h} elements")
        router_scale = router_scale.contiguous()
    return dev, m, h, gate_weight.shape[0], router_scale


def moe_router_logits(x, router_scale, gate_weight, eps: float = 1e-6):
    """Router front-end of GemmaBatchedMoE.forward (gemma.py:75-76) in one launch:
    bf16 logits [M, E] of the gate linear applied to
    router_norm(x) * (router_scale * H**-0.5), with the bf16 roundings of the
    bf16 model (norm output, scaled router_scale, their product, the logits).
    ``router_scale`` may be None (ones); ``gate_weight`` is the nn.Linear weight
    [E, H]."""
    dev, m, h, e, rs = _router_inputs(x, router_scale, gate_weight, "moe_router_logits")
    logits = torch.empty((m, e), dtype=torch.bfloat16, device=dev)
    if m == 0:
        return logits
    L.check(L.load().gi_moe_router_logits(
        _ptr(x.contiguous()), L.DTYPE_BF16, _ptr(rs), _ptr(gate_weight.contiguous()), float(eps),
        _ptr(logits), m, h, e, _stream(dev)), "moe_router_logits")
    return logits


def moe_layer_from_hidden(x, router_scale, gate_weight, gate_up_packed, gate_up_scales,
                          down_packed, down_scales, top_k, group_size, expert_scale=None,
                          eps: float = 1e-6, out=None, *, spin_limit: int = 0):
    """GemmaBatchedMoE.forward (gemma.py:75-98) from the hidden state: the router
    front-end (one launch) feeding ``moe_layer`` on the logits it writes.

    Returns (out [M, H] bf16 -- overwritten, idx int32 [M, top_k],
    weights bf16 [M, top_k], logits bf16 [M, E]).
    """
    dev, m, h, e, rs = _router_inputs(x, router_scale, gate_weight, "moe_layer_from_hidden")
    raise_pending_device_error(dev)
    _on_device(x, gate_up_packed, gate_up_scales, down_packed, down_scales)
    m2, h2, i, e2 = _moe_weight_shapes(x, gate_up_packed, gate_up_scales, down_packed, down_scales)
    _require(e2 == e, f"gate weight has {e} experts, the expert weights {e2}")
    _require(0 < top_k <= min(e, 64), f"top_k must be in [1, min(E, 64)], got {top_k}")
    if expert_scale is not None:
        _on_device(x, expert_scale)
        _require(expert_scale.numel() == e, "expert_scale must have E elements")
        expert_scale = expert_scale.to(torch.float32).contiguous()
    if out is None:
        out = torch.empty_like(x)
    _require(tuple(out.shape) == (m, h) and out.dtype == x.dtype and out.is_contiguous(),
             "out must be a contiguous bf16 [M, H] tensor")
    idx = torch.empty((m, top_k), dtype=torch.int32, device=dev)
    w = torch.empty((m, top_k), dtype=torch.bfloat16, device=dev)
    logits = torch.empty((m, e), dtype=torch.bfloat16, device=dev)
    if m == 0:
        return out, idx, w, logits
    lib = L.load()
    nbytes = lib.gi_fused_moe_workspace_bytes(m, top_k, h, i, e)
    ws = _WS.get("moe", dev, nbytes)
    L.check(lib.gi_moe_layer_from_hidden(
        _ptr(x.contiguous()), L.DTYPE_BF16, _ptr(rs), _ptr(gate_weight.contiguous()), float(eps),
        _ptr(logits), _ptr(expert_scale), _ptr(gate_up_packed), _ptr(gate_up_scales),
        gate_up_scales.shape[1], _ptr(down_packed), _ptr(down_scales), down_scales.shape[1],
        _ptr(out), _ptr(idx), _ptr(w), m, h, i, e, int(top_k), int(group_size), _ptr(ws),
        ws.numel(), int(spin_limit), _stream(dev)), "moe_layer_from_hidden")
    return out, idx, w, logits


def route_topk_softmax(router_logits, top_k, expert_scale=None, out_dtype=torch.bfloat16):
    """idx int32 [M, k], w [M, k] = softmax_fp32(topk(logits)) * expert_scale, cast
    to out_dtype (gemma.py:77-80; ties -> lower expert index)."""
    dev = _on_device(router_logits)
    _require(router_logits.dim() == 2, "router_logits must be [M, E]")
    _require(router_logits.dtype in (torch.bfloat16, torch.float32),
             "router_logits must be bf16 or fp32", TypeError)
    m, e = router_logits.shape
    _require(0 < top_k <= min(e, 64), f"top_k must be in [1, min(E, 64)], got {top_k}")
    if expert_scale is not None:
        _on_device(router_logits, expert_scale)
        expert_scale = expert_scale.to(torch.float32).contiguous()
    idx = torch.empty((m, top_k), dtype=torch.int32, device=dev)
    w = torch.empty((m, top_k), dtype=out_dtype, device=dev)
    logits = router_logits.contiguous()
    L.check(L.load().gi_moe_route_topk_softmax(
        _ptr(logits), _DTYPE_CODE[logits.dtype], _ptr(expert_scale), m, e, int(top_k), _ptr(idx),
        _ptr(w), _DTYPE_CODE[out_dtype], _stream(dev)), "route_topk_softmax")
    return idx, w


def moe_align(expert_indices, num_experts):
    """Token-Union alignment of a [M, top_k] id tensor: dict of unique_experts,
    num_unique, slot_to_unique, offsets, slots (int32 device tensors; entries
    past num_unique are unspecified)."""
    dev = _on_device(expert_indices)
    _require(expert_indices.dim() == 2, "expert_indices must be [M, top_k]")
    m, k = expert_indices.shape
    idx = expert_indices
    if idx.dtype not in (torch.int32, torch.int64):
        idx = idx.to(torch.int32)
    idx = idx.contiguous()
    s = m * k
    umax = min(s, num_experts)
    res = {
        "unique_experts": torch.full((umax,), -1, dtype=torch.int32, device=dev),
        "num_unique": torch.zeros((1,), dtype=torch.int32, device=dev),
        "slot_to_unique": torch.empty((s,), dtype=torch.int32, device=dev),
        "offsets": torch.zeros((umax + 1,), dtype=torch.int32, device=dev),
        "slots": torch.full((s,), -1, dtype=torch.int32, device=dev),
    }
    L.check(L.load().gi_moe_align(
        _ptr(idx), _DTYPE_CODE[idx.dtype], m, k, int(num_experts), _ptr(res["unique_experts"]),
        _ptr(res["num_unique"]), _ptr(res["slot_to_unique"]), _ptr(res["offsets"]),
        _ptr(res["slots"]), _stream(dev)), "moe_align")
    return res


# ---------------------------------------------------------------------------
# W4A16 linear
# ---------------------------------------------------------------------------
def marlin_w4a16(A, B_packed, scales, C, group_size, softcap: float = 0.0):
    """C = A @ dequant(B_packed, scales)  (drop-in for gemmainfer_csrc.marlin_w4a16).

    Overwrites C (reference marlin.cu:704-856).  ``softcap > 0`` fuses the
    final-logit softcap cap*tanh(C/cap) (gemma.py:356-357).
    """
    dev = _on_device(A, B_packed, scales, C)
    _require_act_dtype(A, "marlin_w4a16")
    _require(A.dim() == 2, f"A must be [M, K], got {tuple(A.shape)}")
    m, k = A.shape
    _require(B_packed.dim() == 2 and B_packed.dtype == torch.int32 and B_packed.shape[0] * 8 == k,
             f"B_packed must be int32 [K/8, N] with K={k}, got {tuple(B_packed.shape)}")
    n = B_packed.shape[1]
    _require(scales.dim() == 2 and scales.shape[1] == n and scales.dtype == A.dtype,
             f"scales must be [groups, N={n}] of A's dtype")
    _require(tuple(C.shape) == (m, n) and C.dtype == A.dtype,
             f"C must be [M, N] = {(m, n)} of A's dtype")
    _require(B_packed.is_contiguous() and scales.is_contiguous(), "B_packed/scales must be contiguous")
    _require(isinstance(group_size, int) and group_size > 0 and group_size % 8 == 0,
             f"group_size must be a positive multiple of 8, got {group_size}")
    if m == 0:
        return
    Ac = A.contiguous()
    Cc = C if C.is_contiguous() else torch.empty_like(C, memory_format=torch.contiguous_format)
    lib = L.load()
    nbytes = lib.gi_w4a16_workspace_bytes(m, k, n, group_size)
    ws = _WS.get("w4a16", dev, nbytes) if nbytes else None
    L.check(lib.gi_w4a16_linear(
        _ptr(Ac), _DTYPE_CODE[A.dtype], _ptr(B_packed), _ptr(scales), scales.shape[0], _ptr(Cc), m, k, n,
        int(group_size), float(softcap), _ptr(ws), 0 if ws is None else ws.numel(), _stream(dev)),
        "marlin_w4a16")
    if Cc is not C:
        C.copy_(Cc)


def w4a16_linear(A, B_packed, scales, group_size, softcap: Optional[float] = None):
    """Allocating form of marlin_w4a16; ``softcap`` fuses cap*tanh(y/cap)."""
    C = torch.empty((A.shape[0], B_packed.shape[1]), dtype=A.dtype, device=A.device)
    marlin_w4a16(A, B_packed, scales, C, group_size, softcap=float(softcap or 0.0))
    return C


def _linear_operands(A, B_packed, scales, who):
    _require(B_packed.dim() == 2 and B_packed.dtype == torch.int32 and B_packed.shape[0] * 8 == A.shape[1],
             f"{who}: B_packed must be int32 [K/8, N] with K={A.shape[1]}, got {tuple(B_packed.shape)}")
    _require(scales.dim() == 2 and scales.shape[1] == B_packed.shape[1] and scales.dtype == A.dtype,
             f"{who}: scales must be [groups, N] of A's dtype")
    _require(B_packed.is_contiguous() and scales.is_contiguous(), f"{who}: B_packed/scales must be contiguous")


def w4a16_linear_multi(A, weights, group_size):
    """Several W4A16 projections of the same rows (the q, k, v marlin_w4a16 calls
    of attention.py:115-122) in one grid: one launch, two (the rows' order and
    the products) where the call has enough rows to fill the chip.
    ``weights`` is a list of up to 4 (B_packed, scales); returns the outputs."""
    dev = _on_device(A, *[t for w in weights for t in w])
    _require_bf16(A, "w4a16_linear_multi")
    _require(A.dim() == 2, "A must be [M, K]")
    _require(1 <= len(weights) <= 4, "1 to 4 projections")
    m, k = A.shape
    for B, S in weights:
        _linear_operands(A, B, S, "w4a16_linear_multi")
    outs = [torch.empty((m, B.shape[1]), dtype=A.dtype, device=dev) for B, _ in weights]
    if m == 0:
        return outs
    lib = L.load()
    n = len(weights)
    nbytes = lib.gi_w4a16_linear_multi_workspace_bytes(n, (ctypes.c_int * n)(*[B.shape[1] for B, _ in weights]),
                                                       m, k, int(group_size))
    ws = _WS.get("w4a16", dev, nbytes) if nbytes else None
    arr = lambda vals: (ctypes.c_void_p * n)(*[v.data_ptr() for v in vals])  # noqa: E731
    L.check(lib.gi_w4a16_linear_multi(
        _ptr(A.contiguous()), L.DTYPE_BF16, n, arr([B for B, _ in weights]), arr([S for _, S in weights]),
        (ctypes.c_int * n)(*[S.shape[0] for _, S in weights]), arr(outs),
        (ctypes.c_int * n)(*[B.shape[1] for B, _ in weights]), m, k, int(group_size), _ptr(ws),
        0 if ws is None else ws.numel(), _stream(dev)), "w4a16_linear_multi")
    return outs


def gated_mlp_act(A, gate, up, group_size):
    """GemmaMLP's ``gelu_tanh(gate_proj(x)) * up_proj(x)`` (activations.py:26-28)
    with the bf16 roundings of those torch statements, in one grid as in
    ``w4a16_linear_multi``.  ``gate`` and ``up`` are (B_packed, scales); returns bf16 [M, N]."""
    dev = _on_device(A, *gate, *up)
    _require_bf16(A, "gated_mlp_act")
    _require(A.dim() == 2, "A must be [M, K]")
    _linear_operands(A, *gate, "gated_mlp_act")
    _linear_operands(A, *up, "gated_mlp_act")
    _require(gate[0].shape == up[0].shape, "gate and up projections must have the same shape")
    m, k = A.shape
    n = gate[0].shape[1]
    out = torch.empty((m, n), dtype=A.dtype, device=dev)
    if m == 0:
        return out
    lib = L.load()
    nbytes = lib.gi_w4a16_gated_mlp_workspace_bytes(m, k, n, group_size)
    ws = _WS.get("w4a16", dev, nbytes) if nbytes else None
    L.check(lib.gi_w4a16_gated_mlp(
        _ptr(A.contiguous()), L.DTYPE_BF16, _ptr(gate[0]), _ptr(gate[1]), gate[1].shape[0], _ptr(up[0]),
        _ptr(up[1]), up[1].shape[0], _ptr(out), m, k, n, int(group_size), _ptr(ws),
        0 if ws is None else ws.numel(), _stream(dev)), "gated_mlp_act")
    return out


# ---------------------------------------------------------------------------
# companions
# ---------------------------------------------------------------------------
def softcapping(logits, cap: float):
    dev = _on_device(logits)
    _require(logits.dtype in (torch.bfloat16, torch.float16, torch.float32),
             "softcapping: bf16/fp16/fp32 only", TypeError)
    t = logits if logits.is_contiguous() else logits.contiguous()
    L.check(L.load().gi_softcap_inplace(_ptr(t), _DTYPE_CODE[t.dtype], t.numel(), float(cap),
                                        _stream(dev)), "softcapping")
    if t is not logits:
        logits.copy_(t)


def rmsnorm(input, weight, output, eps: float, add_unit_offset: bool):
    dev = _on_device(input, output)
    _require(input.dtype in (torch.bfloat16, torch.float16, torch.float32),
             "rmsnorm: bf16/fp16/fp32 only", TypeError)
    _require(output.shape == input.shape and output.dtype == input.dtype, "rmsnorm: output mismatch")
    hidden = input.shape[-1]
    x = input.contiguous()
    has_w = weight is not None and weight.numel() > 0
    w = None
    if has_w:
        _on_device(input, weight)
        _require(weight.numel() == hidden, "rmsnorm: weight must have hidden elements")
        w = weight.to(input.dtype).contiguous()
    o = output if output.is_contiguous() else torch.empty_like(output, memory_format=torch.contiguous_format)
    L.check(L.load().gi_rmsnorm(_ptr(x), _ptr(w), _ptr(o), _DTYPE_CODE[x.dtype],
                                x.numel() // hidden if hidden else 0, hidden, float(eps),
                                int(bool(add_unit_offset)), _stream(dev)), "rmsnorm")
    if o is not output:
        output.copy_(o)


def fused_rope_inplace(q, k, cos, sin, position_ids):
    dev = _on_device(q, cos, sin, position_ids)
    _require(q.dim() == 4, "q must be [B, Hq, S, D]")
    _require(q.stride(-1) == 1, "q's last dimension must be contiguous")
    b, hq, s, d = q.shape
    has_k = k is not None and k.numel() > 0
    if has_k:
        _on_device(q, k)
        _require(k.dim() == 4 and k.shape[0] == b and k.shape[2] == s and k.shape[3] == d
                 and k.dtype == q.dtype and k.stride(-1) == 1, "k must be [B, Hk, S, D] like q")
    c = cos.to(q.dtype).contiguous()
    sn = sin.to(q.dtype).contiguous()
    pos = position_ids.to(torch.int64).contiguous()
    _require(pos.numel() == b * s, "position_ids must have B*S elements")
    ks = k.stride()[:3] if has_k else (0, 0, 0)
    L.check(L.load().gi_rope_inplace(
        _ptr(q), _ptr(k) if has_k else None, _ptr(c), _ptr(sn), _ptr(pos), _DTYPE_CODE[q.dtype],
        b, hq, k.shape[1] if has_k else 0, s, d, q.stride(0), q.stride(1), q.stride(2),
        ks[0], ks[1], ks[2], _stream(dev)), "fused_rope_inplace")


# ---------------------------------------------------------------------------
# attention over an 8-bit paged K/V cache
# ---------------------------------------------------------------------------
class KVCache(NamedTuple):
    """A pool of pages of e4m3 codes with one fp32 scale per page and kv head:
    ``k`` [pages, Hk, page, D], ``v`` [pages, Hk, D, page] (transposed),
    ``k_scale`` and ``v_scale`` [pages, Hk]; a value is code * scale."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class KVSlots(NamedTuple):
    """Where a step's rows go (``kv_slots``).  ``status`` is {free pages used
    so far, pages that were lacking, rows dropped}."""
    slots: torch.Tensor      # int64 [rows]
    positions: torch.Tensor  # int64 [rows]
    q_start: torch.Tensor    # int32 [B + 1]
    seq_lens: torch.Tensor   # int32 [B]
    status: torch.Tensor     # int32 [3]


_PAGE_SIZES = (16, 32, 64, 128, 256)
_HEAD_WIDTHS = (64, 128, 256, 512)
_ROW_DTYPES = (torch.bfloat16, torch.float16)
_MAX_COUNT = 0x7fffffff  # rows, requests and table columns are ints of the C entries


# A decode step calls these a few times a layer with kernels of microseconds:
# messages are only formatted where they are raised.
def _launch(device: torch.device, what: str, *args) -> None:
    """gi_``what``(*args, stream).  Kernels are launched on the current device: make it the tensors' own."""
    fn = getattr(L.load(), "gi_" + what)
    if torch.cuda.current_device() == device.index:
        st = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _stream(device))
    if st != L.GI_OK:
        L.check(st, what)


def kv_cache(num_pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> KVCache:
    """An empty cache.  ``page_size`` is 16, 32, 64, 128 or 256 tokens, ``head_dim``
    64, 128, 256 or 512; a token takes 2 * kv_heads * head_dim bytes."""
    _require(num_pages > 0 and kv_heads > 0, "kv_cache: num_pages and kv_heads must be positive")
    _require(page_size in _PAGE_SIZES, f"kv_cache: page_size must be one of {_PAGE_SIZES}, got {page_size}")
    _require(head_dim in _HEAD_WIDTHS, f"kv_cache: head_dim must be one of {_HEAD_WIDTHS}, got {head_dim}")
    codes = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)  # noqa: E731
    scale = lambda: torch.zeros((num_pages, kv_heads), dtype=torch.float32, device=device)  # noqa: E731
    return KVCache(codes(num_pages, kv_heads, page_size, head_dim), codes(num_pages, kv_heads, head_dim, page_size),
                   scale(), scale())


def _cache_shape(cache, who):
    k, v, ks, vs = cache
    if k.dim() != 4:
        raise ValueError(f"{who}: cache.k must be [pages, Hk, page, D], got {tuple(k.shape)}")
    pages, hk, page, d = k.shape
    if v.shape != (pages, hk, d, page):
        raise ValueError(f"{who}: cache.v must be {(pages, hk, d, page)}, got {tuple(v.shape)}")
    if ks.shape != (pages, hk) or vs.shape != (pages, hk):
        raise ValueError(f"{who}: cache scales must be [pages, Hk] = {(pages, hk)}")
    if k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{who}: cache.k and cache.v must be float8_e4m3fn, got {k.dtype} and {v.dtype}")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError(f"{who}: cache scales must be fp32, got {ks.dtype} and {vs.dtype}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{who}: the cache must be contiguous")
    if page not in _PAGE_SIZES:
        raise ValueError(f"{who}: page size must be one of {_PAGE_SIZES}, got {page}")
    return pages, hk, page, d


def _vector(t, dtype, who, name, numel=None):
    if t.dtype != dtype:
        raise TypeError(f"{who}: {name} must be {dtype}, got {t.dtype}")
    if t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous vector")
    if t.numel() > _MAX_COUNT:
        raise ValueError(f"{who}: {name} must have fewer than 2^31 elements, got {t.numel()}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{who}: {name} must have {numel} elements, got {t.numel()}")


def _table(block_table, batch, who):
    if block_table.dtype != torch.int32:
        raise TypeError(f"{who}: block_table must be int32, got {block_table.dtype}")
    if block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError(f"{who}: block_table must be [B={batch}, pages], got {tuple(block_table.shape)}")
    cols, (rs, cs) = block_table.shape[1], block_table.stride()
    if cols > _MAX_COUNT:
        raise ValueError(f"{who}: block_table must have fewer than 2^31 columns, got {cols}")
    if cols > 1 and cs != 1:
        raise ValueError(f"{who}: block_table's rows must be contiguous")
    if batch > 1 and rs < cols:
        raise ValueError(f"{who}: block_table's rows must not overlap")
    return cols, max(rs, cols)


def kv_slots(ctx_lens, new_lens, block_table, free_pages, free_used, page_size, num_rows) -> KVSlots:
    """Places the new tokens of B requests on cache pages, on the device.

    ``ctx_lens``/``new_lens`` int32 [B]: tokens in the cache, tokens to add.
    ``block_table`` int32 [B, max_pages] is written where the step opens pages
    (those from token ceil(ctx / page) * page on, whatever stood there), which
    come from ``free_pages`` (int32) behind the first ``free_used[0]`` of
    them.  ``num_rows`` rows are laid out (the packed rows of q, k and v,
    request after request); those behind the last request get slot -1 and
    position 0.  A row without a page gets slot -1; ``status`` counts what was
    lacking.  Pass ``status`` as the next step's ``free_used``."""
    dev = _on_device(ctx_lens, new_lens, block_table, free_pages, free_used)
    b = ctx_lens.numel()
    _vector(ctx_lens, torch.int32, "kv_slots", "ctx_lens")
    _vector(new_lens, torch.int32, "kv_slots", "new_lens", b)
    _vector(free_pages, torch.int32, "kv_slots", "free_pages")
    _vector(free_used, torch.int32, "kv_slots", "free_used")
    if free_used.numel() < 1:
        raise ValueError("kv_slots: free_used must have an element")
    if page_size not in _PAGE_SIZES:
        raise ValueError(f"kv_slots: page_size must be one of {_PAGE_SIZES}, got {page_size}")
    if not 0 <= num_rows < 2 ** 31:
        raise ValueError(f"kv_slots: num_rows must be in [0, 2^31), got {num_rows}")
    cols, stride = _table(block_table, b, "kv_slots")
    slots, positions = torch.empty((2, num_rows), dtype=torch.int64, device=dev).unbind(0)
    q_start, seq_lens, status = torch.split_with_sizes(torch.empty(2 * b + 4, dtype=torch.int32, device=dev),
                                                       (b + 1, b, 3))
    _launch(dev, "kv_slots",
        ctx_lens.data_ptr(), new_lens.data_ptr(), b, block_table.data_ptr(), cols, stride, free_pages.data_ptr(),
        free_pages.numel(), free_used.data_ptr(), page_size, slots.data_ptr(), positions.data_ptr(), num_rows,
        q_start.data_ptr(), seq_lens.data_ptr(), status.data_ptr())
    return KVSlots(slots, positions, q_start, seq_lens, status)


def rope_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                     original_len: int = 8192, fast: float = 32.0, slow: float = 1.0, device="cuda"):
    """(inv_freq fp64 [rotary_dim / 2], mscale) for ``rope_rows``: base^(-2i / rotary_dim), and for long contexts

    * ``scaling="linear"``: every frequency divided by ``factor``;
    * ``scaling="ntk"``: base * factor^(d / (d - 2)), which leaves the fastest
      frequency and divides the slowest by ``factor``;
    * ``scaling="yarn"``: frequencies that turn more than ``fast`` times in
      ``original_len`` tokens are left, those of fewer than ``slow`` turns are
      divided by ``factor``, with a linear ramp over the turns between (over the turns, not
      over the frequency's index); mscale = 0.1 ln(factor) + 1.
    """
    _require(rotary_dim > 0 and rotary_dim % 2 == 0, f"rope_frequencies: rotary_dim must be even, got {rotary_dim}")
    _require(scaling in (None, "linear", "ntk", "yarn"),
             f"rope_frequencies: scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    _require(base > 0 and factor >= 1, "rope_frequencies: base > 0 and factor >= 1 required")
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    mscale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        _require(fast > slow, "rope_frequencies: fast must be greater than slow")
        turns = original_len * f / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
        mscale = 0.1 * math.log(factor) + 1
    return f.to(device), mscale


def rope_rows(q, k, positions, inv_freq, *, interleaved: bool = False, mscale: float = 1.0, inplace: bool = False):
    """Rotary embedding of packed rows q [T, Hq, D] and k [T, Hk, D] (or None) at
    ``positions`` (int64 [T]); returns the rotated (q, k), which are q and k
    themselves with ``inplace`` (they must not share elements then).

    ``inv_freq`` (fp64, on the device; ``rope_frequencies``) holds one frequency
    per rotated pair: the first 2 * len(inv_freq) dimensions turn, pair i being
    (i, i + len) or, ``interleaved``, (2i, 2i + 1); the others are kept.
    ``mscale`` multiplies cos and sin."""
    dev = _on_device(q, positions, inv_freq) if k is None else _on_device(q, k, positions, inv_freq)
    if q.dtype not in _ACT_DTYPES:
        raise TypeError(f"rope_rows: bf16/fp16/fp32 only, got {q.dtype}")
    if q.dim() != 3:
        raise ValueError(f"rope_rows: q must be [T, Hq, D], got {tuple(q.shape)}")
    t, hq, d = q.shape
    qs = q.stride()
    if qs[2] != 1 and d > 1:
        raise ValueError("rope_rows: q's last dimension must be contiguous")
    hk, ks = 0, (0, 0)
    if k is not None:
        if k.dim() != 3 or k.shape[0] != t or k.shape[2] != d or k.dtype != q.dtype:
            raise ValueError(f"rope_rows: k must be [{t}, Hk, {d}] of q's dtype, got {tuple(k.shape)} {k.dtype}")
        hk, ks = k.shape[1], k.stride()
        if ks[2] != 1 and d > 1:
            raise ValueError("rope_rows: k's last dimension must be contiguous")
    _vector(positions, torch.int64, "rope_rows", "positions", t)
    _vector(inv_freq, torch.float64, "rope_rows", "inv_freq")
    rot = 2 * inv_freq.numel()
    if not 0 < rot <= d:
        raise ValueError(f"rope_rows: {inv_freq.numel()} frequencies rotate {rot} of {d} dimensions")
    if inplace:
        qo, ko, qos, kos = q, k, qs, ks
        for name, x in (("q", q), ("k", k)):
            if x is not None and _broadcast(x):
                raise ValueError(f"rope_rows: {name} has broadcast dimensions, which cannot be rotated in place")
        if k is not None and k.data_ptr() == q.data_ptr() and k.numel() and q.numel():
            raise ValueError("rope_rows: q and k are the same elements, which cannot both be rotated in place")
    else:
        qo = torch.empty((t, hq, d), dtype=q.dtype, device=dev)
        qos = (hq * d, d)
        ko = None if k is None else torch.empty((t, hk, d), dtype=q.dtype, device=dev)
        kos = (hk * d, d)
    if t == 0:
        return qo, ko
    _launch(dev, "rope_rows",
        q.data_ptr(), qo.data_ptr(), None if k is None else k.data_ptr(), None if k is None else ko.data_ptr(),
        positions.data_ptr(), inv_freq.data_ptr(), _DTYPE_CODE[q.dtype], t, hq, hk, d, rot, bool(interleaved),
        mscale, qs[0], qs[1], qos[0], qos[1], ks[0], ks[1], kos[0], kos[1])
    return qo, ko


def kv_append(k, v, slots, cache: KVCache) -> None:
    """Stores rows k and v [T, Hk, D] (bf16/fp16/fp32) in the cache at ``slots``
    (int64 [T]; negative ones, and those past the last page, are skipped).

    The rows of one page must follow each other, as those of a request do
    (skipped rows may stand between them); of rows with the same slot the last
    one is stored.  Each page has one scale per
    head for K and one for V, a power of two that grows as larger rows arrive
    (what the page holds is then rounded to the new one); writing a page's first
    place starts the page anew.  A row with an infinity or NaN makes its page's
    scale NaN until then."""
    dev = _on_device(k, v, slots, *cache)
    pages, hk, page, d = _cache_shape(cache, "kv_append")
    if k.dtype not in _ACT_DTYPES or v.dtype != k.dtype:
        raise TypeError(f"kv_append: k and v must be bf16, fp16 or fp32, alike; got {k.dtype} and {v.dtype}")
    t = slots.numel()
    if k.shape != (t, hk, d) or v.shape != k.shape:
        raise ValueError(f"kv_append: k and v must be [{t}, {hk}, {d}] (one row a slot), got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError("kv_append: the last dimension of k and v must be contiguous")
    _vector(slots, torch.int64, "kv_append", "slots")
    _launch(dev, "kv_append",
        k.data_ptr(), v.data_ptr(), _DTYPE_CODE[k.dtype], ks[0], ks[1], vs[0], vs[1], slots.data_ptr(), t, hk, d,
        page, pages, cache[0].data_ptr(), cache[1].data_ptr(), cache[2].data_ptr(), cache[3].data_ptr())


def _rows_aligned(x):
    s = x.stride()
    return s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and x.data_ptr() % 16 == 0


def _broadcast(x):
    return any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape))


def _overlap(x, y):
    """Whether the bytes that two tensors span meet (a tensor's own gaps count as its)."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a, b), (c, d) = span(x), span(y)
    return x.numel() > 0 and y.numel() > 0 and a < d and c < b


def kv_attention(q, cache: KVCache, block_table, seq_lens, q_start=None, *, scale: Optional[float] = None,
                 window: int = 0, out=None):
    """Causal attention of packed query rows q [T, Hq, D] (bf16 or fp16) over the
    cache; returns [T, Hq, D].

    Rows ``q_start[b]`` to ``q_start[b + 1]`` (int32 [B + 1], which must not
    decrease; None: one row a request) are the last tokens of request b, which has ``seq_lens[b]`` (int32)
    tokens in the pages ``block_table[b]`` names, those rows' own among them.  A
    row sees the tokens up to its own, with ``window`` > 0 the last ``window`` of
    them; one that sees none gets zeros.  ``scale`` defaults to D ** -0.5.  Query
    head h reads kv head h // (Hq // Hk).  ``out`` is like q, its rows contiguous
    and 16-byte aligned, and overlaps neither what q spans nor itself.  Rows behind the last request are not
    computed: they keep what ``out`` holds, and are unspecified without it.  A
    row that sees a token without a page (one outside the cache) gets NaN, and so
    does every row of a request that is longer than its table."""
    if q_start is None:
        dev = _on_device(q, block_table, seq_lens, *cache)
    else:
        dev = _on_device(q, block_table, seq_lens, q_start, *cache)
    pages, hk, page, d = _cache_shape(cache, "kv_attention")
    if q.dtype not in _ROW_DTYPES:
        raise TypeError(f"kv_attention: q must be bf16 or fp16, got {q.dtype}")
    if q.dim() != 3 or q.shape[2] != d or q.shape[1] % hk or q.shape[1] == 0:
        raise ValueError(f"kv_attention: q must be [T, a multiple of {hk}, {d}], got {tuple(q.shape)}")
    if d not in _HEAD_WIDTHS:
        raise ValueError(f"kv_attention: head width must be one of {_HEAD_WIDTHS}, got {d}")
    t, hq, _ = q.shape
    if t > _MAX_COUNT:
        raise ValueError(f"kv_attention: fewer than 2^31 rows, got {t}")
    b = seq_lens.numel()
    _vector(seq_lens, torch.int32, "kv_attention", "seq_lens")
    cols, stride = _table(block_table, b, "kv_attention")
    if q_start is not None:
        _vector(q_start, torch.int32, "kv_attention", "q_start", b + 1)
    elif t != b:
        raise ValueError(f"kv_attention: without q_start there is one row a request: {t} rows, {b} requests")
    if window < 0:
        raise ValueError(f"kv_attention: window must be >= 0 (0: none), got {window}")
    window = min(window, _MAX_COUNT)  # what the C entry's int holds; no table is that long
    if out is None:
        out = torch.empty((t, hq, d), dtype=q.dtype, device=dev)
        os = (hq * d, d)
    else:
        _on_device(q, out)
        if out.shape != q.shape or out.dtype != q.dtype or not _rows_aligned(out):
            raise ValueError("kv_attention: out must be like q, its rows contiguous and 16-byte aligned")
        if _overlap(q, out):
            raise ValueError("kv_attention: out must not overlap q")
        if _broadcast(out):
            raise ValueError("kv_attention: out has broadcast dimensions, whose rows would be written together")
        os = out.stride()
    if t == 0 or b == 0:
        return out
    if not _rows_aligned(q):
        q = q.clone(memory_format=torch.contiguous_format)
    qs = q.stride()
    lib = L.load()
    nbytes = lib.gi_kv_attention_workspace_bytes(t, b, hq, hk, d, cols * page)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(dev, "kv_attention",
        q.data_ptr(), _DTYPE_CODE[q.dtype], qs[0], qs[1], cache[0].data_ptr(), cache[1].data_ptr(),
        cache[2].data_ptr(), cache[3].data_ptr(), block_table.data_ptr(), cols, stride, seq_lens.data_ptr(),
        None if q_start is None else q_start.data_ptr(), out.data_ptr(), os[0], os[1], t, b, hq, hk, d, page,
        pages, d ** -0.5 if scale is None else scale, window, ws.data_ptr(), nbytes)
    return out
