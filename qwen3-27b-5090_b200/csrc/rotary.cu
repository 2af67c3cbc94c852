// Queries and keys between their projection and the attention: per-head RMS norm (optional), rotation by position, and
// the write of keys and values into the paged cache, in one pass over the projection's rows.
//
// Mathematics. A head x of D channels becomes
//   n = x / sqrt(mean(x^2) + eps) * (1 + w)  (or * w; or n = x without the norm),
//   pairs (n_a, n_b) of the first rot channels -> amplitude * (n_a cos t - n_b sin t, n_a sin t + n_b cos t), t = pos w_i,
// with the pairs (i, i + rot/2) or, interleaved, (2i, 2i + 1); channels past rot keep their values.
//
// The angle. Only pos * w_i modulo a whole turn matters, and at position 10^6 an fp32 product has lost 0.06 rad of it. So
// w_i is kept as a 64-bit binary fraction of a turn and multiplied by the position in integers: the product modulo 2^64
// IS the angle modulo a turn, with an error of |pos| 2^-65 turns, for negative positions too. The nearest quarter turn is
// taken off in integers as well; what is left, at most an eighth of a turn, is rounded to fp32 once (2^-24 relative).
//
// Bound: memory (every value is read and written once). Shape: a CTA takes a few tokens; its threads first compute the
// (token, pair) table of cos and sin once into shared memory - not once per head, which would cost more instructions
// than the loads leave room for - and then walk the tokens' head rows, D / 8 lanes to a row, 8 channels (4 pairs) to a lane.
//
// Programmatic dependent launch: as every kernel of this library, wait for the predecessor first, release the successor
// only then.
#include <cmath>
#include <cuda_fp16.h>

#include "../../include/q27b200/capi.h"
#include "common.cuh"
#include "ptx_sm100.cuh"

namespace q27b {
namespace {

using Args = q27b_qk_rope;

constexpr int kThreads = 256;

// Four consecutive channels.
__device__ __forceinline__ void load4(const float* p, float* v) {
  const float4 t = *reinterpret_cast<const float4*>(p);
  v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float* v) {
  const uint2 t = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(t.x << 16), v[1] = __uint_as_float(t.x & 0xFFFF0000u);
  v[2] = __uint_as_float(t.y << 16), v[3] = __uint_as_float(t.y & 0xFFFF0000u);
}
__device__ __forceinline__ void load4(const __half* p, float* v) {
  const uint2 t = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&t.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
// The one rounding of a result to its type (nearest even).
__device__ __forceinline__ void store4(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* v) {
  __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}
__device__ __forceinline__ void store4(__half* p, const float* v) {
  __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}

// cos and sin of a binary fraction of a turn, times the amplitude.
__device__ __forceinline__ float2 cos_sin_turn(uint64_t turn, float amplitude) {
  const uint64_t shifted = turn + (uint64_t(1) << 61);             // + 1/8 turn: the top two bits are the nearest quarter
  const int64_t rest = int64_t(turn - (shifted & (uint64_t(3) << 62)));  // within +- 1/8 turn
  float s, c;
  sincospif(float(rest) * 0x1p-63f, &s, &c);  // (the fraction of a HALF turn: rest 2^-64 turns)
  const uint32_t quarter = uint32_t(shifted >> 62);
  const float c1 = (quarter & 1u) ? -s : c, s1 = (quarter & 1u) ? c : s;  // + 1/4 turn: (cos, sin) -> (-sin, cos)
  const float sign = (quarter & 2u) ? -amplitude : amplitude;
  return make_float2(c1 * sign, s1 * sign);
}

template <typename W>
__device__ __forceinline__ void load_weight(const W* w, int at, bool zero_centred, float* v) {
  load4(w + at, v);
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = zero_centred ? 1.f + v[i] : v[i];
}

template <typename In, typename Out, int kLanes>
__global__ void __launch_bounds__(kThreads) qk_rope_kernel(const __grid_constant__ Args p, int tokens, uint32_t* status) {
  extern __shared__ float2 table[];  // [tokens of this CTA][rot / 2] (cos, sin)
  pdl_wait();
  pdl_trigger();
  const int t0 = blockIdx.x * tokens, nt = min(tokens, p.T - t0), pairs = p.rot_dim / 2;
  for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
    const int t = t0 + i / pairs;
    const int64_t pos = p.pos64 ? static_cast<const int64_t*>(p.positions)[t] : int64_t(static_cast<const int32_t*>(p.positions)[t]);
    table[i] = cos_sin_turn(uint64_t(pos) * p.turns[i % pairs], p.amplitude);
  }
  const int lane = threadIdx.x % kLanes, D = p.head_dim;
  const bool active = lane * 8 < D, turns = lane * 8 < p.rot_dim;
  int a, b;  // the two groups of four channels of this lane
  if (p.interleaved || !turns)
    a = lane * 8, b = a + 4;
  else
    a = lane * 4, b = pairs + lane * 4;
  float wq[8], wk[8];
  const bool norm = p.q_weight != nullptr;
  if (norm && active) {
    if (p.weight_f32) {
      load_weight(static_cast<const float*>(p.q_weight), a, p.zero_centred, wq), load_weight(static_cast<const float*>(p.q_weight), b, p.zero_centred, wq + 4);
      load_weight(static_cast<const float*>(p.k_weight), a, p.zero_centred, wk), load_weight(static_cast<const float*>(p.k_weight), b, p.zero_centred, wk + 4);
    } else {
      using B = __nv_bfloat16;
      load_weight(static_cast<const B*>(p.q_weight), a, p.zero_centred, wq), load_weight(static_cast<const B*>(p.q_weight), b, p.zero_centred, wq + 4);
      load_weight(static_cast<const B*>(p.k_weight), a, p.zero_centred, wk), load_weight(static_cast<const B*>(p.k_weight), b, p.zero_centred, wk + 4);
    }
  }
  __syncthreads();

  const int vheads = p.v ? p.k_heads : 0, rows = p.q_heads + p.k_heads + vheads;
  const int step = (kThreads / kLanes) * gridDim.y;
  const float inv_dim = 1.f / float(D);  // exact or rounded once: D <= 256
  // grid.y shares the rows of a token group out when there are few tokens
  // (the loop runs the same number of times in every lane of a warp: the shuffles below are whole-warp)
  const int total = nt * rows;
  for (int r0 = blockIdx.y * (kThreads / kLanes); r0 < total; r0 += step) {
    const int r = r0 + threadIdx.x / kLanes;
    const bool live = active && r < total;
    const int tl = live ? r / rows : 0, t = t0 + tl;
    int head = live ? r - tl * rows : 0;
    const int kind = head < p.q_heads ? 0 : head < p.q_heads + p.k_heads ? 1 : 2;
    head -= kind == 0 ? 0 : kind == 1 ? p.q_heads : p.q_heads + p.k_heads;
    float x[8] = {};
    if (live) {
      const In* src = kind == 0 ? static_cast<const In*>(p.q) + t * p.q_ld_token + head * p.q_ld_head
                    : kind == 1 ? static_cast<const In*>(p.k) + t * p.k_ld_token + head * p.k_ld_head
                                : static_cast<const In*>(p.v) + t * p.v_ld_token + head * p.v_ld_head;
      load4(src + a, x), load4(src + b, x + 4);
    }
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (kind < 2) {
        const float rms = rsqrtf(ss * inv_dim + p.eps);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] *= rms * (kind == 0 ? wq[i] : wk[i]);
      }
    }
    if (!live) continue;
    if (kind < 2 && turns) {
      const float2* cs = table + tl * pairs + lane * 4;
      if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 e = cs[i];
          const float u = x[2 * i], v = x[2 * i + 1];
          x[2 * i] = u * e.x - v * e.y, x[2 * i + 1] = u * e.y + v * e.x;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 e = cs[i];
          const float u = x[i], v = x[i + 4];
          x[i] = u * e.x - v * e.y, x[i + 4] = u * e.y + v * e.x;
        }
      }
    }
    Out* dst;
    if (kind == 0) {
      dst = static_cast<Out*>(p.q_out) + t * p.q_out_ld_token + head * p.q_out_ld_head;
    } else if (p.slots) {
      const int64_t slot = p.slots[t];
      if (slot < 0) continue;  // a padding token: nothing is written
      const int64_t page = slot / p.page_size, at = slot - page * p.page_size;
      if (page >= p.pages) {  // no such place in the cache
        atomicCAS(status, 0u, uint32_t(kStatusBadSlot));
        continue;
      }
      dst = kind == 1 ? static_cast<Out*>(p.k_cache) + page * p.kc_ld_page + head * p.kc_ld_head + at * p.kc_ld_slot
                      : static_cast<Out*>(p.v_cache) + page * p.vc_ld_page + head * p.vc_ld_head + at * p.vc_ld_slot;
    } else {
      dst = static_cast<Out*>(p.k_out) + t * p.k_out_ld_token + head * p.k_out_ld_head;
    }
    store4(dst + a, x), store4(dst + b, x + 4);
  }
}

size_t type_size(int dtype) { return dtype == Q27B_F32 ? 4 : 2; }

template <typename In, typename Out, int kLanes>
int launch(const Args& p, cudaStream_t s) {
  const int rows = p.q_heads + p.k_heads + (p.v ? p.k_heads : 0), groups = kThreads / kLanes;
  const int sms = sm_count();
  // Many tokens: four to a CTA, so that the cos / sin table costs one evaluation per thread. Few: one to a CTA, and its
  // rows shared out over grid.y until the CTAs fill the GPU.
  const int tokens = p.T >= 4 * 8 * sms ? 4 : 1;
  const int blocks = (p.T + tokens - 1) / tokens;
  int share = 1;
  while (blocks * share * 2 <= 2 * sms && share * 2 * groups <= rows + groups - 1) share *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(blocks), unsigned(share)), cfg.blockDim = dim3(kThreads), cfg.stream = s;
  cfg.dynamicSmemBytes = size_t(tokens) * (p.rot_dim / 2) * sizeof(float2);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 1 : 0;
  uint32_t* status = device_status_ptr();
  Q27B_REQUIRE(status, "qk_rope: no device status word");
  Q27B_CUDA(cudaLaunchKernelEx(&cfg, qk_rope_kernel<In, Out, kLanes>, p, tokens, status));
  return 0;
}

template <typename In, typename Out>
int launch_lanes(const Args& p, cudaStream_t s) {
  if (p.head_dim <= 64) return launch<In, Out, 8>(p, s);
  if (p.head_dim <= 128) return launch<In, Out, 16>(p, s);
  return launch<In, Out, 32>(p, s);
}

template <typename In>
int launch_out(const Args& p, cudaStream_t s) {
  if (p.out_dtype == Q27B_F32) return launch_lanes<In, float>(p, s);
  if (p.out_dtype == Q27B_BF16) return launch_lanes<In, __nv_bfloat16>(p, s);
  return launch_lanes<In, __half>(p, s);
}

// A tensor whose rows are loaded and stored four channels at a time: base and strides in whole groups of four.
bool grouped(const void* base, int dtype, int64_t ld0, int64_t ld1, int64_t ld2 = 0) {
  return base && (reinterpret_cast<uintptr_t>(base) % (4 * type_size(dtype))) == 0 && ld0 % 4 == 0 && ld1 % 4 == 0 && ld2 % 4 == 0;
}

}  // namespace
}  // namespace q27b

using namespace q27b;

extern "C" {

int q27b_rope_turns(int rot_dim, double base, int scaling, double factor, double original_len, double beta_fast, double beta_slow,
                    uint64_t* turns, float* amplitude) {
  Q27B_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && turns && amplitude, "rope_turns: rot_dim must be positive and even, outputs not null");
  Q27B_REQUIRE(std::isfinite(base) && base > 1.0, "rope_turns: the base must be finite and above 1");
  Q27B_REQUIRE(scaling >= 0 && scaling <= 3, "rope_turns: scaling must be 0 (none), 1 (linear), 2 (ntk) or 3 (yarn)");
  Q27B_REQUIRE(scaling == 0 || (std::isfinite(factor) && factor >= 1.0), "rope_turns: the factor must be finite and at least 1");
  Q27B_REQUIRE(scaling != 2 || rot_dim > 2, "rope_turns: ntk scaling needs more than one pair");
  Q27B_REQUIRE(scaling != 3 || (std::isfinite(original_len) && original_len > 0 && std::isfinite(beta_fast) && beta_slow > 0 && beta_fast > beta_slow),
               "rope_turns: yarn needs the original length and beta_fast > beta_slow > 0");
  const long double tau = 2.0L * std::acos(-1.0L);
  long double b = base;
  if (scaling == 2) b *= std::pow((long double)factor, (long double)rot_dim / (rot_dim - 2));
  for (int i = 0; i < rot_dim / 2; i++) {
    long double w = std::pow(b, -2.0L * i / rot_dim) / tau;  // turns per position, at most 1 / (2 pi)
    if (scaling == 1) w /= factor;
    if (scaling == 3) {
      const long double r = (original_len * w - beta_slow) / ((long double)beta_fast - beta_slow);
      const long double keep = r < 0 ? 0.0L : r > 1 ? 1.0L : r;
      w = w * keep + w / factor * (1 - keep);
    }
    turns[i] = uint64_t(std::roundl(std::ldexp(w, 64)));
  }
  *amplitude = scaling == 3 ? float(0.1 * std::log(factor) + 1.0) : 1.f;
  return 0;
}

int q27b_qk_norm_rope(const q27b_qk_rope* a, void* stream) {
  Q27B_REQUIRE(a, "qk_norm_rope: null arguments");
  const Args& p = *a;
  Q27B_REQUIRE(p.T >= 0 && p.q_heads > 0 && p.k_heads >= 0 && p.q_heads <= 4096 && p.k_heads <= 4096,
               "qk_norm_rope: bad counts (T = %d, heads = %d and %d)", p.T, p.q_heads, p.k_heads);
  Q27B_REQUIRE(p.head_dim > 0 && p.head_dim % 8 == 0 && p.head_dim <= 256, "qk_norm_rope: head_dim must be a multiple of 8 up to 256 (%d)", p.head_dim);
  Q27B_REQUIRE(p.rot_dim > 0 && p.rot_dim % 8 == 0 && p.rot_dim <= p.head_dim, "qk_norm_rope: rot_dim must be a multiple of 8 up to head_dim (%d)", p.rot_dim);
  Q27B_REQUIRE(p.in_dtype >= 0 && p.in_dtype <= 2 && p.out_dtype >= 0 && p.out_dtype <= 2, "qk_norm_rope: unknown type");
  if (p.T == 0) return 0;
  Q27B_REQUIRE(p.positions && p.turns, "qk_norm_rope: null positions or frequencies");
  Q27B_REQUIRE(grouped(p.q, p.in_dtype, p.q_ld_token, p.q_ld_head) && grouped(p.q_out, p.out_dtype, p.q_out_ld_token, p.q_out_ld_head),
               "qk_norm_rope: q and q_out must not be null and must start and stride in whole groups of four channels");
  Q27B_REQUIRE(!p.q_weight == !p.k_weight || p.k_heads == 0, "qk_norm_rope: the norm needs both weights");
  if (p.q_weight) {
    const int wt = p.weight_f32 ? Q27B_F32 : Q27B_BF16;
    Q27B_REQUIRE(grouped(p.q_weight, wt, 0, 0) && (p.k_heads == 0 || grouped(p.k_weight, wt, 0, 0)), "qk_norm_rope: the weights must be aligned to four values");
    Q27B_REQUIRE(p.eps >= 0.f, "qk_norm_rope: eps must not be negative");
  }
  Q27B_REQUIRE(p.k_heads > 0 || (!p.k && !p.v && !p.slots), "qk_norm_rope: keys, values or slots without key heads");
  if (p.k_heads > 0) {
    Q27B_REQUIRE(grouped(p.k, p.in_dtype, p.k_ld_token, p.k_ld_head), "qk_norm_rope: k must not be null and must start and stride in whole groups of four channels");
    Q27B_REQUIRE(!p.v || (p.slots && grouped(p.v, p.in_dtype, p.v_ld_token, p.v_ld_head)),
                 "qk_norm_rope: v goes into the cache only, and must start and stride in whole groups of four channels");
    if (p.slots) {
      Q27B_REQUIRE(!p.k_out, "qk_norm_rope: keys go either to k_out or into the cache");
      Q27B_REQUIRE(p.page_size > 0 && p.pages > 0 && grouped(p.k_cache, p.out_dtype, p.kc_ld_page, p.kc_ld_head, p.kc_ld_slot) &&
                       (!p.v || grouped(p.v_cache, p.out_dtype, p.vc_ld_page, p.vc_ld_head, p.vc_ld_slot)),
                   "qk_norm_rope: the cache must not be null or empty and must start and stride in whole groups of four channels");
    } else {
      Q27B_REQUIRE(grouped(p.k_out, p.out_dtype, p.k_out_ld_token, p.k_out_ld_head),
                   "qk_norm_rope: k_out must not be null and must start and stride in whole groups of four channels");
    }
  }
  Args c = p;
  if (c.q_weight && !c.k_weight) c.k_weight = c.q_weight;  // (no key heads: loaded, not used)
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.in_dtype == Q27B_F32) return launch_out<float>(c, s);
  if (p.in_dtype == Q27B_BF16) return launch_out<__nv_bfloat16>(c, s);
  return launch_out<__half>(c, s);
}

}  // extern "C"
