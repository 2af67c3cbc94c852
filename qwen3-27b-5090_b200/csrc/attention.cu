// Attention of the newest tokens of a batch of sequences over a paged key / value cache, with an optional sliding window
// and sink tokens.
//
// Mathematics. Row i of a sequence with n new rows and L tokens stands at position p = L - n + i and sees the keys
// j <= p with j > p - window or j < sinks. With s_j = scale q . k_j:  o = sum_j exp(s_j - m) v_j / l,  l = sum_j exp(s_j - m),
// m the running maximum: one pass over the keys, in fp32.
#include <algorithm>
#include <cmath>

#include <cuda.h>
#include <cuda_fp16.h>

#include "../../include/q27b200/capi.h"
#include "common.cuh"
#include "ptx_sm100.cuh"

namespace q27b {
namespace {

using Args = q27b_attention;

__device__ __forceinline__ float2 widen(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 widen(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ void narrow(float2 v, __nv_bfloat162* o) { *o = __float22bfloat162_rn(v); }
__device__ __forceinline__ void narrow(float2 v, __half2* o) { *o = __float22half2_rn(v); }

// Rows and length of sequence b, cut to what exists: rows to [0, T], the length to what the table can name (positions
// still count from the full length).
struct Sequence {
  int row0, rows, len, reach;  // reach: keys [0, reach) have a table entry
};
__device__ __forceinline__ Sequence sequence_of(const Args& p, int b) {
  Sequence s;
  s.row0 = b, s.rows = 1;
  if (p.q_begin) {
    s.row0 = min(max(p.q_begin[b], 0), p.T);
    s.rows = min(max(p.q_begin[b + 1], s.row0), p.T) - s.row0;
  }
  s.len = max(p.kv_lens[b], 0);
  s.reach = int(min(int64_t(s.len), int64_t(p.table_width) * p.page_size));
  return s;
}

// One row's result from its sums: D / N channels by each of N threads, 1 / l applied and rounded once; thread 0 the lse.
template <typename T2, int D, int N>
__device__ __forceinline__ void store_row(const Args& p, int t, int head, int part, float m, float l, const float* src) {
  constexpr int E = D / N >= 8 ? 8 : D / N;
  const bool some = !(l == 0.f);  // (NaN counts as something)
  const float inv = some ? 1.f / l : 0.f;
  uint16_t* out = static_cast<uint16_t*>(p.out) + t * p.out_ld_token + head * p.out_ld_head;
#pragma unroll
  for (int k = 0; k < D / (N * E); k++) {
    const int d = (k * N + part) * E;
    T2 w[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; e++) narrow(make_float2(src[d + 2 * e] * inv, src[d + 2 * e + 1] * inv), &w[e]);
    if constexpr (E == 8)
      *reinterpret_cast<uint4*>(out + d) = *reinterpret_cast<uint4*>(w);
    else if constexpr (E == 4)
      *reinterpret_cast<uint2*>(out + d) = *reinterpret_cast<uint2*>(w);
    else
      *reinterpret_cast<uint32_t*>(out + d) = *reinterpret_cast<uint32_t*>(w);
  }
  if (p.lse && part == 0) p.lse[int64_t(t) * p.heads + head] = some ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

// ---- tensor maps -----------------------------------------------------------------------------------------------------

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// Keys or values as (channel, token in page, head, page), copied in boxes of 64 channels x `box` tokens with the 128-byte
// swizzle; a page outside the cache reads as zeros.
int make_cache_map(CUtensorMap* map, const Args& p, const void* cache, int64_t ld_page, int64_t ld_head, int64_t ld_slot, int box) {
  EncodeTiledFn fn = encode_fn();
  Q27B_REQUIRE(fn, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[4] = {cuuint64_t(p.head_dim), cuuint64_t(p.page_size), cuuint64_t(p.kv_heads), cuuint64_t(p.pages)};
  const cuuint64_t row = cuuint64_t(p.head_dim) * 2;  // (the stride of a dimension of one is never used)
  const cuuint64_t strides[3] = {cuuint64_t(ld_slot) * 2, p.kv_heads > 1 ? cuuint64_t(ld_head) * 2 : row, p.pages > 1 ? cuuint64_t(ld_page) * 2 : row};
  const cuuint32_t boxes[4] = {64u, cuuint32_t(box), 1u, 1u}, estr[4] = {1u, 1u, 1u, 1u};
  const CUresult r = fn(map, p.dtype == Q27B_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(cache),
                        dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  Q27B_REQUIRE(r == CUDA_SUCCESS, "attention: cuTensorMapEncodeTiled failed (%d) for cache strides %lld, %lld, %lld", int(r), (long long)ld_page,
               (long long)ld_head, (long long)ld_slot);
  return 0;
}

#include "attention_stream.inl"
#include "attention_tile.inl"

// Which kernels a call needs: sequences of up to kStreamRows query rows per key head stream, longer ones go through the tensor
// cores' 128-row tiles. The host knows the rows only through the hint, so whichever kernels it picks take every sequence between
// them: a kernel that is alone takes all.
struct Choice {
  bool stream, tile;
};
Choice choose(const Args& p) {
  const int64_t rows = int64_t(p.q_begin ? std::min(p.max_new, p.T) : 1) * (p.heads / p.kv_heads);
  const bool tile = rows > kStreamRows;
  return {!tile || (p.B > 1 && p.heads / p.kv_heads <= kStreamRows && p.q_begin), tile};
}

template <typename T2, int D>
int run(const Args& p, cudaStream_t s) {
  uint32_t* status = device_status_ptr();
  Q27B_REQUIRE(status, "attention: no device status word");
  const Choice c = choose(p);
  if (c.stream)
    if (int rc = launch_stream<T2, D>(p, c.tile ? kStreamRows : 1 << 30, p.ws, s, status)) return rc;
  if (c.tile) return launch_tile<T2, D>(p, c.stream ? kStreamRows + 1 : 1, p.ws, s, status);
  return 0;
}

template <typename T2>
int run_dim(const Args& p, cudaStream_t s) {
  if (p.head_dim == 64) return run<T2, 64>(p, s);
  if (p.head_dim == 128) return run<T2, 128>(p, s);
  return run<T2, 256>(p, s);
}

// (the two kernels of a mixed call run one after the other: they share the scratch)
template <int D>
size_t scratch_bytes_of(const Args& p) {
  const Choice c = choose(p);
  const int sms = sm_count();
  return std::max(c.stream ? stream_scratch_bytes<D>(StreamCfg<D>::kCtasPerSm * sms) : size_t(0), c.tile ? tile_scratch_bytes<D>(sms) : size_t(0));
}
size_t scratch_bytes(const Args& p) {
  if (p.head_dim == 64) return scratch_bytes_of<64>(p);
  if (p.head_dim == 128) return scratch_bytes_of<128>(p);
  return scratch_bytes_of<256>(p);
}

int check_sizes(const Args& p) {
  Q27B_REQUIRE(p.dtype == Q27B_BF16 || p.dtype == Q27B_F16, "attention: the type must be bf16 or fp16");
  Q27B_REQUIRE(p.B >= 0 && p.T >= 0 && p.B <= (1 << 20), "attention: bad counts (B = %d, T = %d)", p.B, p.T);
  Q27B_REQUIRE(p.heads > 0 && p.kv_heads > 0 && p.heads <= 4096 && p.heads % p.kv_heads == 0,
               "attention: heads must be a positive multiple of kv_heads (%d, %d)", p.heads, p.kv_heads);
  Q27B_REQUIRE(p.head_dim == 64 || p.head_dim == 128 || p.head_dim == 256, "attention: head_dim must be 64, 128 or 256 (%d)", p.head_dim);
  Q27B_REQUIRE(p.page_size == 16 || p.page_size == 32 || p.page_size == 64 || p.page_size == 128,
               "attention: page_size must be 16, 32, 64 or 128 (%d)", p.page_size);
  Q27B_REQUIRE(p.pages > 0 && p.table_width > 0 && int64_t(p.table_width) * p.page_size < (int64_t(1) << 30),
               "attention: the cache and the table must not be empty, nor the table name 2^30 tokens or more (pages = %d, width = %d)", p.pages, p.table_width);
  Q27B_REQUIRE(int64_t(p.T) * p.heads < (int64_t(1) << 30), "attention: T x heads must stay below 2^30 (%d, %d)", p.T, p.heads);
  Q27B_REQUIRE(p.window >= 0 && p.sinks >= 0, "attention: window and sinks must not be negative");
  Q27B_REQUIRE(p.scale >= 0.f && p.scale < INFINITY, "attention: the scale must be finite and not negative (%g)", double(p.scale));
  Q27B_REQUIRE(p.max_new >= 1 && p.max_kv >= 1, "attention: max_new and max_kv must be at least 1");
  return 0;
}

// 16-byte base and strides (in elements).
bool rows16(const void* base, int64_t a, int64_t b, int64_t c = 0) { return base && aligned16(base) && a % 8 == 0 && b % 8 == 0 && c % 8 == 0; }

}  // namespace
}  // namespace q27b

using namespace q27b;

extern "C" {

int q27b_attention_workspace(const q27b_attention* a, size_t* bytes) {
  Q27B_REQUIRE(a && bytes, "attention_workspace: null arguments");
  if (int rc = check_sizes(*a)) return rc;
  *bytes = a->T == 0 || a->B == 0 ? 0 : scratch_bytes(*a);
  return 0;
}

int q27b_paged_attention(const q27b_attention* a, void* stream) {
  Q27B_REQUIRE(a, "attention: null arguments");
  Args p = *a;
  if (int rc = check_sizes(p)) return rc;
  if (p.T == 0 || p.B == 0) return 0;
  Q27B_REQUIRE(p.q_begin || p.T == p.B, "attention: without q_begin there is one row per sequence (T = %d, B = %d)", p.T, p.B);
  Q27B_REQUIRE(p.table && p.kv_lens, "attention: null table or lengths");
  Q27B_REQUIRE(rows16(p.q, p.q_ld_token, p.q_ld_head) && rows16(p.out, p.out_ld_token, p.out_ld_head),
               "attention: q and out must not be null, 16-byte aligned, with strides that are multiples of 8 elements");
  Q27B_REQUIRE(rows16(p.k_cache, p.kc_ld_page, p.kc_ld_head, p.kc_ld_slot) && rows16(p.v_cache, p.vc_ld_page, p.vc_ld_head, p.vc_ld_slot),
               "attention: the cache must not be null, 16-byte aligned, with strides that are multiples of 8 elements");
  Q27B_REQUIRE((p.kv_heads == 1 || (p.kc_ld_head > 0 && p.vc_ld_head > 0)) && (p.pages == 1 || (p.kc_ld_page > 0 && p.vc_ld_page > 0)) && p.kc_ld_slot > 0 && p.vc_ld_slot > 0,
               "attention: the cache's strides must be positive");
  const size_t need = scratch_bytes(p);
  Q27B_REQUIRE(p.ws && (reinterpret_cast<uintptr_t>(p.ws) & 255u) == 0 && p.ws_bytes >= need, "attention: needs %zu bytes of 256-byte aligned scratch, got %zu", need, p.ws_bytes);
  if (p.window >= (1 << 30)) p.window = 0;  // (no table names a position that far)
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p.dtype == Q27B_BF16 ? run_dim<__nv_bfloat162>(p, s) : run_dim<__half2>(p, s);
}

}  // extern "C"
