"""Queries and keys between their projection and the attention (q27b_qk_norm_rope): rotation by position, alone or fused
with the per-head RMS norm and with the write of keys and values into the paged cache. Every call is one launch on
torch's current stream of the tensors' device; nothing synchronises, and a call may be captured into a CUDA graph.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from .q27lib import call

SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # Q27B_F32, Q27B_BF16, Q27B_F16
# q27b_qk_rope (include/q27b200/capi.h), field by field
QK_ROPE = struct.Struct("@11i2f" + "PPPP" + "Pqq" * 5 + "P2i" + "Pqqq" * 2)
_NONE3 = (0, 0, 0)


def device_of(what: str, *tensors: torch.Tensor) -> torch.device:
    """The one CUDA device all the tensors are on; None entries are skipped."""
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"{what}: tensors must be on a CUDA device, got one on {dev}")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: all tensors must be on one device, got {dev} and {t.device}")
    return dev


def launch(name: str, packed: bytes, dev: torch.device):
    """The C entry on the device's current stream; the device is made current for the call where it is not."""
    if dev.index == torch.cuda.current_device():
        call(name, packed, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            call(name, packed, torch.cuda.current_stream(dev).cuda_stream)


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


def _heads(what: str, x: torch.Tensor, T: int, D: int, heads: int | None = None):
    if x.dim() != 3 or x.shape[0] != T or x.shape[2] != D or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{what}: expected [{T}, {'heads' if heads is None else heads}, {D}], got {list(x.shape)}")
    if x.stride(2) != 1 and D > 1:
        raise ValueError(f"{what}: the channels of a head must be contiguous")


def _launch(what, rotary, positions, q, k, v, q_out, k_out, q_weight, k_weight, eps, zero_centred, cache, slots):
    if q.dim() != 3:
        raise ValueError(f"{what}: q must be [tokens, heads, channels], got {list(q.shape)}")
    T, Hq, D = q.shape
    dev = device_of(what, q, positions, rotary.turns, k, v, q_out, k_out, q_weight, k_weight, slots, cache.k if cache else None)
    _heads(what + ": q", q, T, D)
    if q.dtype not in DTYPES:
        raise ValueError(f"{what}: q must be fp32, bf16 or fp16, got {q.dtype}")
    if positions.dtype not in (torch.int64, torch.int32) or positions.shape != (T,) or not positions.is_contiguous():
        raise ValueError(f"{what}: positions must be int64 or int32 [{T}], contiguous")
    Hk = 0
    if k is not None:
        Hk = k.shape[1] if k.dim() == 3 else 0
        _heads(what + ": k", k, T, D)
        if v is not None:
            _heads(what + ": v", v, T, D, Hk)
        if any(x is not None and x.dtype != q.dtype for x in (k, v)):
            raise ValueError(f"{what}: q, k and v must have one type")
    _heads(what + ": q_out", q_out, T, D, Hq)
    if q_weight is not None:
        if q_weight.dtype not in (torch.float32, torch.bfloat16) or any(w is not None and (w.dtype != q_weight.dtype or w.shape != (D,) or not w.is_contiguous()) for w in (q_weight, k_weight)):
            raise ValueError(f"{what}: the norm weights must be fp32 or bf16 [{D}], contiguous, of one type")
    ko = kc = vc = None
    page_size = pages = 0
    if cache is not None:
        if slots is None or slots.dtype != torch.int64 or slots.shape != (T,) or not slots.is_contiguous():
            raise ValueError(f"{what}: slots must be int64 [{T}], contiguous")
        if cache.kv_heads != Hk or cache.head_dim != D or cache.k.dtype != q_out.dtype:
            raise ValueError(f"{what}: the cache holds {cache.kv_heads} heads of {cache.head_dim} channels in {cache.k.dtype}, got {Hk} of {D} for {q_out.dtype}")
        kc, vc = cache.k_packed, cache.v_packed
        page_size, pages = cache.page_size, cache.pages
    elif k is not None:
        _heads(what + ": k_out", k_out, T, D, Hk)
        if k_out.dtype != q_out.dtype:
            raise ValueError(f"{what}: q_out and k_out must have one type")
        ko = (k_out.data_ptr(), k_out.stride(0), k_out.stride(1))
    if q_out.dtype not in DTYPES:
        raise ValueError(f"{what}: outputs must be fp32, bf16 or fp16, got {q_out.dtype}")
    packed = QK_ROPE.pack(
        T, Hq, Hk, D, rotary.rot_dim, rotary.interleaved, DTYPES[q.dtype], DTYPES[q_out.dtype], positions.dtype == torch.int64,
        q_weight is not None and q_weight.dtype == torch.float32, zero_centred, eps, rotary.amplitude,
        positions.data_ptr(), rotary.turns.data_ptr(), 0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
        q.data_ptr(), q.stride(0), q.stride(1),
        *(_NONE3 if k is None else (k.data_ptr(), k.stride(0), k.stride(1))),
        *(_NONE3 if v is None else (v.data_ptr(), v.stride(0), v.stride(1))),
        q_out.data_ptr(), q_out.stride(0), q_out.stride(1), *(ko or _NONE3),
        0 if cache is None else slots.data_ptr(), page_size, pages, *(kc or (0, 0, 0, 0)), *(vc or (0, 0, 0, 0)))
    launch("q27b_qk_norm_rope", packed, dev)


def rope(rotary: Rotary, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
         k_out: torch.Tensor | None = None):
    """Rotates q [T, heads, D] (and k [T, kv_heads, D]) by positions [T]; returns (q_out, k_out). The outputs may be the inputs
    themselves; without them new tensors of the inputs' type are made."""
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
    if k is not None and k_out is None:
        k_out = torch.empty(k.shape, dtype=q_out.dtype, device=k.device)
    _launch("rope", rotary, positions, q, k, None, q_out, k_out, None, None, 0.0, False, None, None)
    return q_out, k_out


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
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=cache.k.dtype if cache is not None else dtype or q.dtype, device=q.device)
    if cache is None and k_out is None:
        k_out = torch.empty(k.shape, dtype=q_out.dtype, device=k.device)
    _launch("qk_norm_rope", rotary, positions, q, k, v, q_out, k_out, q_weight, k_weight, float(eps), zero_centred, cache, slots)
    return q_out if cache is not None else (q_out, k_out)
