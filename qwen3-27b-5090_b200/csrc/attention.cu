// Attention of the newest tokens of a batch of sequences over a paged key / value cache, with an optional sliding window
// and sink tokens.
//
// Mathematics. Row i of a sequence with n new rows and L tokens stands at position p = L - n + i and sees the keys
// j <= p with j > p - window or j < sinks. With s_j = scale q . k_j:  o = sum_j exp(s_j - m) v_j / l,  l = sum_j exp(s_j - m),
// m the running maximum: one pass over the keys, in fp32.
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

// One warp per (row, head), keys one after the other.
template <typename T2, int D>
__global__ void __launch_bounds__(128) attention_row_kernel(const __grid_constant__ Args p, uint32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int64_t w = int64_t(blockIdx.x) * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (w >= int64_t(p.T) * p.heads) return;
  const int t = int(w / p.heads), h = int(w % p.heads), hk = h / (p.heads / p.kv_heads);
  int b = t;
  if (p.q_begin) {  // the last b with q_begin[b] <= t
    int lo = 0, hi = p.B;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (p.q_begin[mid] <= t) lo = mid + 1; else hi = mid;
    }
    b = lo - 1;
  }
  if (b < 0 || b >= p.B) return;
  const Sequence s = sequence_of(p, b);
  if (t < s.row0 || t >= s.row0 + s.rows) return;
  const int pos = s.len - s.rows + (t - s.row0);
  constexpr int E = D / 64;  // channel pairs per lane
  using Pair = T2;
  float2 q[E], o[E];
  const Pair* qp = reinterpret_cast<const Pair*>(static_cast<const uint16_t*>(p.q) + t * p.q_ld_token + h * p.q_ld_head);
#pragma unroll
  for (int e = 0; e < E; e++) q[e] = widen(qp[lane + 32 * e]), o[e] = make_float2(0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  const int low = p.window > 0 ? max(pos - p.window + 1, 0) : 0;
  const int end = min(pos + 1, s.reach);
  if (pos + 1 > s.reach && lane == 0) atomicCAS(status, 0u, uint32_t(kStatusBadPage));
  for (int j = 0; j < end; j++) {
    if (j >= p.sinks && j < low) {
      j = low - 1;
      continue;
    }
    const int page = p.table[b * p.table_ld + j / p.page_size];
    if (page < 0 || page >= p.pages) {
      if (lane == 0) atomicCAS(status, 0u, uint32_t(kStatusBadPage));
      continue;
    }
    const int at = j % p.page_size;
    const Pair* kp = reinterpret_cast<const Pair*>(static_cast<const uint16_t*>(p.k_cache) + page * p.kc_ld_page + hk * p.kc_ld_head + at * p.kc_ld_slot);
    const Pair* vp = reinterpret_cast<const Pair*>(static_cast<const uint16_t*>(p.v_cache) + page * p.vc_ld_page + hk * p.vc_ld_head + at * p.vc_ld_slot);
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float2 k = widen(kp[lane + 32 * e]);
      d = fmaf(q[e].x, k.x, fmaf(q[e].y, k.y, d));
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
    d *= p.scale;
    const float m2 = fmaxf(m, d), keep = expf(m - m2), pr = expf(d - m2);
    m = m2, l = l * keep + pr;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float2 v = widen(vp[lane + 32 * e]);
      o[e].x = o[e].x * keep + pr * v.x, o[e].y = o[e].y * keep + pr * v.y;
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  Pair* op = reinterpret_cast<Pair*>(static_cast<uint16_t*>(p.out) + t * p.out_ld_token + h * p.out_ld_head);
#pragma unroll
  for (int e = 0; e < E; e++) narrow(make_float2(o[e].x * inv, o[e].y * inv), &op[lane + 32 * e]);
  if (p.lse && lane == 0) p.lse[w] = l > 0.f || l != l ? m + logf(l) : -INFINITY;
}

template <typename T2, int D>
int launch_rows(const Args& p, cudaStream_t s) {
  uint32_t* status = device_status_ptr();
  Q27B_REQUIRE(status, "attention: no device status word");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((int64_t(p.T) * p.heads + 3) / 4)), cfg.blockDim = dim3(128), cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 1 : 0;
  Q27B_CUDA(cudaLaunchKernelEx(&cfg, attention_row_kernel<T2, D>, p, status));
  return 0;
}

template <typename T2>
int launch_dim(const Args& p, cudaStream_t s) {
  if (p.head_dim == 64) return launch_rows<T2, 64>(p, s);
  if (p.head_dim == 128) return launch_rows<T2, 128>(p, s);
  return launch_rows<T2, 256>(p, s);
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
  Q27B_REQUIRE(p.window >= 0 && p.sinks >= 0, "attention: window and sinks must not be negative");
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
  *bytes = 0;
  return 0;
}

int q27b_paged_attention(const q27b_attention* a, void* stream) {
  Q27B_REQUIRE(a, "attention: null arguments");
  const Args& p = *a;
  if (int rc = check_sizes(p)) return rc;
  if (p.T == 0 || p.B == 0) return 0;
  Q27B_REQUIRE(p.q_begin || p.T == p.B, "attention: without q_begin there is one row per sequence (T = %d, B = %d)", p.T, p.B);
  Q27B_REQUIRE(p.table && p.kv_lens, "attention: null table or lengths");
  Q27B_REQUIRE(rows16(p.q, p.q_ld_token, p.q_ld_head) && rows16(p.out, p.out_ld_token, p.out_ld_head),
               "attention: q and out must not be null, 16-byte aligned, with strides that are multiples of 8 elements");
  Q27B_REQUIRE(rows16(p.k_cache, p.kc_ld_page, p.kc_ld_head, p.kc_ld_slot) && rows16(p.v_cache, p.vc_ld_page, p.vc_ld_head, p.vc_ld_slot),
               "attention: the cache must not be null, 16-byte aligned, with strides that are multiples of 8 elements");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p.dtype == Q27B_BF16 ? launch_dim<__nv_bfloat162>(p, s) : launch_dim<__half2>(p, s);
}

}  // extern "C"
