"""Queries and keys between their projection and the attention (q27b_qk_norm_rope): rotation by position, alone or fused
with the per-head RMS norm and with the write of keys and values into the paged cache. Every call is one launch on
torch's current stream of the tensors' device; nothing synchronises, and a call may be captured into a CUDA graph.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from .q27lib import call, last_error, lib

SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # Q27B_F32, Q27B_BF16, Q27B_F16
# q27b_qk_rope (include/q27b200/capi.h), field by field
QK_ROPE = struct.Struct("@11i2f" + "PPPP" + "Pqq" * 5 + "P2i" + "Pqqq" * 2)
_NONE3, _NONE4 = (0, 0, 0), (0, 0, 0, 0)


def device_of(what: str, *tensors: torch.Tensor) -> torch.device:
    """The one CUDA device all the tensors are on; None entries are skipped."""
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"{what}: tensors must be on a CUDA device, got one on {dev}")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: all tensors must be on one device, got {dev} and {t.device}")
    return dev


_entries: dict = {}


def launch(name: str, packed: bytes, dev: torch.device):
    """The C entry on the device's current stream; the device is made current for the call where it is not."""
    index = dev.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return launch(name, packed, dev)
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(lib(), name)
    # (the raw handle: making a Stream object of it costs as much as the launch)
    if fn(packed, torch._C._cuda_getCurrentRawStream(index)):
        raise RuntimeError(f"{name}: {last_error()}")


class Rotary:
    """The rotation of one model's heads: speeds of the rot_dim / 2 channel pairs as binary fractions of a turn (on the
    device) and the factor on cos and sin. The first rot_dim channels of a head turn, in pairs (i, i + rot_dim / 2) or,
    interleaved, (2 i, 2 i + 1). scaling stretches the speeds for contexts `factor` times the trained original_len: "linear",
    "ntk" (the base raised) or "yarn" (Peng et al. 2023), whose amplitude 0.1 ln(factor) + 1 `amplitude` overrides."""

    def __init__(self, rot_dim: int, base: float = 10000.0, interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
                 original_len: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0, amplitude: float | None = None,
                 device="cuda"):
        if scaling not in SCALINGS:
            raise ValueError(f"Rotary: scaling must be one of {', '.join(SCALINGS)}, got {scaling!r}")
        self.rot_dim, self.interleaved = rot_dim, bool(interleaved)
        turns, a = (ctypes.c_uint64 * max(rot_dim // 2, 1))(), ctypes.c_float()
        call("q27b_rope_turns", rot_dim, base, SCALINGS[scaling], factor, original_len, beta_fast, beta_slow, turns, ctypes.byref(a))
        self.amplitude = float(a.value if amplitude is None else amplitude)
        signed = [t - (1 << 64) if t >> 63 else t for t in turns]
        self.turns = torch.tensor(signed, dtype=torch.int64, device=device)
        self.turns_ptr = self.turns.data_ptr()


def _heads(what: str, x: torch.Tensor, shape):
    """Base and strides of [T, heads, D] with contiguous channels."""
    if x.shape != shape:
        raise ValueError(f"{what}: expected {list(shape)}, got {list(x.shape)}")
    a, b, c = x.stride()
    if c != 1 and shape[2] > 1:
        raise ValueError(f"{what}: the channels of a head must be contiguous")
    return x.data_ptr(), a, b


def _launch(what, rotary, positions, q, k, v, q_out, k_out, q_weight, k_weight, eps, zero_centred, cache, slots, out_dtype):
    """Checks, outputs where none are given (of out_dtype), and the launch."""
    if q.dim() != 3 or (k is not None and k.dim() != 3):
        raise ValueError(f"{what}: q and k must be [tokens, heads, channels]")
    shape = q.shape
    T, Hq, D = shape
    dev = device_of(what, q, positions, rotary.turns, k, v, q_out, k_out, q_weight, k_weight, slots, cache.k if cache else None)
    dtype, pos_dtype = q.dtype, positions.dtype
    if q_out is not None:
        out_dtype = q_out.dtype
    in_code, out_code = DTYPES.get(dtype), DTYPES.get(out_dtype)
    if in_code is None or out_code is None:
        raise ValueError(f"{what}: inputs and outputs must be fp32, bf16 or fp16, got {dtype} and {out_dtype}")
    pos64 = pos_dtype is torch.int64
    if not (pos64 or pos_dtype is torch.int32) or positions.shape != (T,) or not positions.is_contiguous():
        raise ValueError(f"{what}: positions must be int64 or int32 [{T}], contiguous")
    qp = _heads(what + ": q", q, shape)
    if q_out is None:
        q_out = torch.empty_like(q, dtype=out_dtype, memory_format=torch.contiguous_format)
        qo = (q_out.data_ptr(), Hq * D, D)
    else:
        qo = _heads(what + ": q_out", q_out, shape)
    Hk, kp, vp, ko = 0, _NONE3, _NONE3, _NONE3
    if k is not None:
        Hk = k.shape[1]
        k_shape = (T, Hk, D)
        kp = _heads(what + ": k", k, k_shape)
        if v is not None:
            vp = _heads(what + ": v", v, k_shape)
        if k.dtype is not dtype or (v is not None and v.dtype is not dtype):
            raise ValueError(f"{what}: q, k and v must have one type")
    qw = kw = 0
    weight_f32 = False
    if q_weight is not None:
        weight_f32 = q_weight.dtype is torch.float32
        if not (weight_f32 or q_weight.dtype is torch.bfloat16) or any(w.dtype is not q_weight.dtype or w.shape != (D,) or not w.is_contiguous() for w in (q_weight, k_weight)):
            raise ValueError(f"{what}: the norm weights must be fp32 or bf16 [{D}], contiguous, of one type")
        qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
    slot_ptr, page_size, pages, kc, vc = 0, 0, 0, _NONE4, _NONE4
    if cache is not None:
        if slots is None or slots.dtype is not torch.int64 or slots.shape != (T,) or not slots.is_contiguous():
            raise ValueError(f"{what}: slots must be int64 [{T}], contiguous")
        if cache.kv_heads != Hk or cache.head_dim != D or cache.dtype is not out_dtype:
            raise ValueError(f"{what}: the cache holds {cache.kv_heads} heads of {cache.head_dim} channels in {cache.dtype}, got {Hk} of {D} for {out_dtype}")
        slot_ptr, page_size, pages, kc, vc = slots.data_ptr(), cache.page_size, cache.pages, cache.k_packed, cache.v_packed
    elif k is not None:
        if k_out is None:
            k_out = torch.empty_like(k, dtype=out_dtype, memory_format=torch.contiguous_format)
            ko = (k_out.data_ptr(), Hk * D, D)
        else:
            ko = _heads(what + ": k_out", k_out, k_shape)
            if k_out.dtype is not out_dtype:
                raise ValueError(f"{what}: q_out and k_out must have one type")
    launch("q27b_qk_norm_rope", QK_ROPE.pack(
        T, Hq, Hk, D, rotary.rot_dim, rotary.interleaved, in_code, out_code, pos64, weight_f32, zero_centred, eps,
        rotary.amplitude, positions.data_ptr(), rotary.turns_ptr, qw, kw, *qp, *kp, *vp, *qo, *ko, slot_ptr, page_size, pages, *kc, *vc), dev)
    return q_out, k_out


def rope(rotary: Rotary, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
         k_out: torch.Tensor | None = None, v: torch.Tensor | None = None, cache=None, slots: torch.Tensor | None = None):
    """Rotates q [T, heads, D] (and k [T, kv_heads, D]) by positions [T]; returns (q_out, k_out). The outputs may be the inputs
    themselves; without them new tensors of the inputs' type are made. With a cache (attention.KvCache) k, and v as it is, go to
    its places slots [T] as in qk_norm_rope, the outputs have its type, and q_out alone is returned."""
    if cache is not None and (k is None or k_out is not None):
        raise ValueError("rope: with a cache k goes into it, and nowhere else")
    if cache is None and (v is not None or slots is not None):
        raise ValueError("rope: v and slots need a cache")
    out = _launch("rope", rotary, positions, q, k, v, q_out, k_out, None, None, 0.0, False, cache, slots, q.dtype if cache is None else cache.dtype)
    return out if cache is None else out[0]


def qk_norm_rope(rotary: Rotary, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 eps: float = 1e-6, zero_centred: bool = True, v: torch.Tensor | None = None, cache=None, slots: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None, dtype: torch.dtype | None = None):
    """x / rms(x) * (1 + weight) per head (zero_centred, as the hidden-size norm of this package; else * weight), then the
    rotation. With a cache (attention.KvCache) the keys, and v as it is, go to its places slots [T] (page * page_size + offset; negative: not
    written; each at most once) and q_out is returned; without one (q_out, k_out). Outputs have the cache's type, else
    `dtype`, else q's. q, k and v may be views of the stacked projection's rows."""
    if cache is not None and k_out is not None:
        raise ValueError("qk_norm_rope: keys go either into the cache or to k_out")
    if cache is None and (v is not None or slots is not None):
        raise ValueError("qk_norm_rope: v and slots need a cache")
    if q_weight is None or k_weight is None or k is None:
        raise ValueError("qk_norm_rope: k and both weights are needed (rope rotates without the norm)")
    out = _launch("qk_norm_rope", rotary, positions, q, k, v, q_out, k_out, q_weight, k_weight, float(eps), zero_centred, cache, slots,
                  cache.dtype if cache is not None else dtype or q.dtype)
    return out if cache is None else out[0]
