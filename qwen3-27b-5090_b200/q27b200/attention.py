"""Attention over a paged key / value cache (q27b_paged_attention), between the q | k | v and the output projection: one
token per sequence, a few (verification), prompt chunks and whole prompts, ragged and mixed in one call; grouped queries; an
optional sliding window with sink tokens. Calls run on torch's current stream of the tensors' device, synchronise nothing and
may be captured into a CUDA graph; lengths, tables and rows may then change from replay to replay.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from .q27lib import call
from .rotary import DTYPES, device_of, launch

# q27b_attention (include/q27b200/capi.h), field by field
ATTENTION = struct.Struct("@13if" + "qPPP" + "Pqq" + "Pqqq" * 2 + "Pqq" + "PPN")


class KvCache:
    """Keys and values of all sequences in pages: k and v [pages, kv_heads, page_size, head_dim], bf16 or fp16. Any strides
    (a view of one combined tensor, or of pages kept token by token, transposed) that leave the channels contiguous and are
    multiples of 8 elements."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError(f"KvCache: k and v must be [pages, kv_heads, page_size, head_dim] of one type and device, got {list(k.shape)} and {list(v.shape)}")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("KvCache: the channels of a head must be contiguous")
        if k.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"KvCache: the type must be bf16 or fp16, got {k.dtype}")
        self.k, self.v, self.dtype = k, v, k.dtype
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.k_packed = (k.data_ptr(), *k.stride()[:3])
        self.v_packed = (v.data_ptr(), *v.stride()[:3])

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, dtype=torch.bfloat16, device="cuda"):
        shape = (pages, kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))

    def slots(self, table: torch.Tensor, sequence: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """Places of tokens in the cache for qk_norm_rope: token i is at positions[i] of sequence[i], a row of the block table. A
        table entry that is negative gives a negative place, which is not written."""
        page = table[sequence.long(), (positions // self.page_size).long()].long()
        return page * self.page_size + positions.long() % self.page_size


class Attention:
    """softmax(scale q k^T) v with the mask of one kind of layer. A token at position p sees the positions j <= p with
    j > p - window (no window: all) or j < sinks. scale: head_dim ** -0.5 unless given."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, window: int | None = None, sinks: int = 0, scale: float | None = None):
        if window is not None and window < 1:
            raise ValueError(f"Attention: the window must be at least 1 (None: no window), got {window}")
        if sinks < 0:
            raise ValueError(f"Attention: sinks must not be negative, got {sinks}")
        if kv_heads < 1 or heads < 1 or heads % kv_heads:
            raise ValueError(f"Attention: heads must be a positive multiple of kv_heads, got {heads} and {kv_heads}")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.window, self.sinks = window or 0, sinks
        self.scale = float(head_dim ** -0.5 if scale is None else scale)

    def __call__(self, q: torch.Tensor, cache: KvCache, table: torch.Tensor, kv_lens: torch.Tensor, q_begin: torch.Tensor | None = None,
                 max_new: int | None = None, max_kv: int | None = None, out: torch.Tensor | None = None,
                 lse: torch.Tensor | None = None) -> torch.Tensor:
        """q [T, heads, head_dim]: the newest tokens of B sequences, whose keys and values are in the cache already. table
        int32 [B, width]: the pages of each sequence in order (entries of pages that no row sees may be anything); kv_lens int32 [B]:
        tokens in the cache, the new ones among them; q_begin int32 [B + 1]: rows of each sequence, None for one row each. max_new,
        max_kv: the longest sequence's rows and length as far as the host knows them; they only steer the split of the work.
        lse: an fp32 [T, heads] tensor that receives ln sum exp(scale q k). Rows in no sequence are not written."""
        if q.dim() != 3 or q.shape[1] != self.heads or q.shape[2] != self.head_dim:
            raise ValueError(f"attention: q must be [T, {self.heads}, {self.head_dim}], got {list(q.shape)}")
        T, B = q.shape[0], kv_lens.shape[0]
        dev = device_of("attention", q, cache.k, table, kv_lens, q_begin, out, lse)
        dtype = q.dtype
        if cache.kv_heads != self.kv_heads or cache.head_dim != self.head_dim or cache.dtype is not dtype:
            raise ValueError(f"attention: the cache holds {cache.kv_heads} heads of {cache.head_dim} channels in {cache.dtype}, the layer has {self.kv_heads} of {self.head_dim} and q is {dtype}")
        if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != B or (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError(f"attention: the table must be int32 [{B}, width] with contiguous rows")
        if kv_lens.dtype is not torch.int32 or kv_lens.dim() != 1 or not kv_lens.is_contiguous():
            raise ValueError("attention: kv_lens must be int32 [B], contiguous")
        if q_begin is not None and (q_begin.dtype is not torch.int32 or q_begin.shape != (B + 1,) or not q_begin.is_contiguous()):
            raise ValueError(f"attention: q_begin must be int32 [{B + 1}], contiguous")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype is not dtype:
            raise ValueError(f"attention: out must be {list(q.shape)} in {dtype}")
        if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (T, self.heads) or not lse.is_contiguous()):
            raise ValueError(f"attention: lse must be fp32 [{T}, {self.heads}], contiguous")
        q0, q1, q2 = q.stride()
        o0, o1, o2 = out.stride()
        if q2 != 1 or o2 != 1:
            raise ValueError("attention: the channels of q and out must be contiguous")
        width = table.shape[1]
        if max_new is None:
            max_new = 1 if q_begin is None else T
        if max_kv is None:
            max_kv = width * cache.page_size
        head = (DTYPES.get(dtype, -1), B, T, self.heads, self.kv_heads, self.head_dim, cache.page_size, cache.pages, width, self.window, self.sinks,
                max(int(max_new), 1), max(int(max_kv), 1), self.scale, table.stride(0), table.data_ptr(), kv_lens.data_ptr(),
                0 if q_begin is None else q_begin.data_ptr(), q.data_ptr(), q0, q1, *cache.k_packed, *cache.v_packed,
                out.data_ptr(), o0, o1, 0 if lse is None else lse.data_ptr())
        if dev.index != torch.cuda.current_device():
            with torch.cuda.device(dev):
                self._run(head, q, dev)
        else:
            self._run(head, q, dev)
        return out

    @staticmethod
    def _run(head, q, dev):
        need = ctypes.c_size_t()
        call("q27b_attention_workspace", ATTENTION.pack(*head, 0, 0), ctypes.byref(need))
        # scratch of this call alone: torch's allocator keeps it apart from other streams' calls and other graphs' replays
        ws = q.new_empty(need.value, dtype=torch.uint8) if need.value else None
        launch("q27b_paged_attention", ATTENTION.pack(*head, 0 if ws is None else ws.data_ptr(), need.value), dev)
