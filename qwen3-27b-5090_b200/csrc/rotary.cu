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
// than the loads leave room for - and then walk the tokens' head rows, D / 16 lanes to a row, 16 channels (8 pairs) to a lane,
// the next row's loads in flight. Measured: 8191 tokens of 28 heads x 256 channels (fp16): 43 us, 5.5 TB/s (84 % of the measured
// copy rate); 4096 tokens of 40 + 8 + 8 heads x 128 channels with the norm into the cache: 26 us, 4.5 TB/s (its 1024 CTAs
// are 1.7 waves of the GPU); with 8 channels to a lane 60 and 44 us; with three or five CTAs per SM instead of four 48 and
// 51, 31 and 33 us; with one token per CTA instead of four 64 and 46 us.
//
// Programmatic dependent launch: as every kernel of this library, wait for the predecessor first, release the successor
// only then.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include <cuda_fp16.h>

#include "../../include/q27b200/capi.h"
#include "common.cuh"
#include "ptx_sm100.cuh"

namespace q27b {
namespace {

using Args = q27b_qk_rope;

constexpr int kThreads = 256, kMostTokens = 4;

// kUnit consecutive channels as they lie in memory, and widened.
template <typename E, int kUnit>
struct Raw {
  static constexpr int kBytes = kUnit * int(sizeof(E)), kVectors = kBytes > 16 ? kBytes / 16 : 1;
  uint4 v[kVectors];  // (8 bytes: the lower half)
  __device__ __forceinline__ void load(const E* p) {
    if constexpr (kBytes == 8) {
      const uint2 t = *reinterpret_cast<const uint2*>(p);
      v[0].x = t.x, v[0].y = t.y;
    } else {
#pragma unroll
      for (int i = 0; i < kVectors; i++) v[i] = reinterpret_cast<const uint4*>(p)[i];
    }
  }
  __device__ __forceinline__ void widen(float* x) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
#pragma unroll
    for (int i = 0; i < kUnit; i++) {
      if constexpr (sizeof(E) == 4)
        x[i] = __uint_as_float(w[i]);
      else if constexpr (std::is_same<E, __nv_bfloat16>::value)
        x[i] = __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
      else
        x[i] = __half2float(__ushort_as_half(uint16_t(i % 2 ? w[i / 2] >> 16 : w[i / 2])));
    }
  }
};
// The one rounding of a result to its type (nearest even).
template <int kUnit>
__device__ __forceinline__ void store(float* p, const float* v) {
#pragma unroll
  for (int i = 0; i < kUnit; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int kUnit, typename Out>
__device__ __forceinline__ void store(Out* p, const float* v) {
  uint32_t w[kUnit / 2];
#pragma unroll
  for (int i = 0; i < kUnit / 2; i++) {
    if constexpr (std::is_same<Out, __nv_bfloat16>::value) {
      __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&t);
    } else {
      __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&t);
    }
  }
  if constexpr (kUnit == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
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

__device__ __forceinline__ void turn_pair(float& a, float& b, float2 cs) {
  const float u = a * cs.x - b * cs.y;
  b = a * cs.y + b * cs.x, a = u;
}

// kLanes lanes to a row, kUnit * 2 channels (kUnit pairs, or two runs that do not turn) to a lane; `tokens` tokens to a CTA.
template <typename In, typename Out, int kUnit, int kLanes>
__global__ void __launch_bounds__(kThreads, 4) qk_rope_kernel(const __grid_constant__ Args p, int tokens, uint32_t* status) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int D = p.head_dim, pairs = p.rot_dim / 2, t0 = blockIdx.x * tokens, nt = min(tokens, p.T - t0);
  float2* table = reinterpret_cast<float2*>(smem);                   // [tokens][pairs] (cos, sin)
  float* weights = reinterpret_cast<float*>(table + tokens * pairs);  // [2][D] what q and k are multiplied by (with the norm)
  __shared__ int64_t place_of[kMostTokens];
  const bool norm = p.q_weight != nullptr;
  pdl_wait();
  pdl_trigger();
  // The CTA's row groups are dealt out to its tokens; a group walks the heads of its token (q, then k, then v).
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, per_token = kThreads / kLanes / tokens;
  const int tl = group / per_token, t = t0 + tl, step = per_token * gridDim.y;
  const int qk_heads = p.q_heads + p.k_heads, rows = qk_heads + (p.v ? p.k_heads : 0);
  const bool active = lane * 2 * kUnit < D && tl < nt, turns = lane * 2 * kUnit < p.rot_dim;
  int a, b;  // the two runs of kUnit channels of this lane
  if (p.interleaved || !turns)
    a = lane * 2 * kUnit, b = a + kUnit;
  else
    a = lane * kUnit, b = pairs + lane * kUnit;
  auto source = [&](int head) {
    return head < p.q_heads ? static_cast<const In*>(p.q) + t * p.q_ld_token + head * p.q_ld_head
           : head < qk_heads ? static_cast<const In*>(p.k) + t * p.k_ld_token + (head - p.q_heads) * p.k_ld_head
                             : static_cast<const In*>(p.v) + t * p.v_ld_token + (head - qk_heads) * p.v_ld_head;
  };
  Raw<In, kUnit> next[2];
  int head = blockIdx.y * per_token + group % per_token;  // (the first row is on its way while the tables are made)
  if (active && head < rows) next[0].load(source(head) + a), next[1].load(source(head) + b);
  for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
    const int t = t0 + i / pairs;
    const int64_t pos = p.pos64 ? static_cast<const int64_t*>(p.positions)[t] : int64_t(static_cast<const int32_t*>(p.positions)[t]);
    table[i] = cos_sin_turn(uint64_t(pos) * p.turns[i % pairs], p.amplitude);
  }
  if (norm)
    for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
      const void* w = i < D ? p.q_weight : p.k_weight;
      const int d = i < D ? i : i - D;
      const float v = p.weight_f32 ? static_cast<const float*>(w)[d] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[d]);
      weights[i] = p.zero_centred ? 1.f + v : v;
    }
  if (p.slots && threadIdx.x < nt) {  // the tokens' places in the cache: page and offset, -1: not written
    const int64_t slot = p.slots[t0 + threadIdx.x], page = slot < 0 ? -1 : slot / p.page_size;
    if (page >= p.pages) atomicCAS(status, 0u, uint32_t(kStatusBadSlot));
    place_of[threadIdx.x] = page < 0 || page >= p.pages ? -1 : (page << 32) | (slot - page * p.page_size);
  }
  __syncthreads();

  float2 cs[kUnit];
  if (active && turns) {
#pragma unroll
    for (int i = 0; i < kUnit; i++) cs[i] = table[tl * pairs + lane * kUnit + i];
  }
  const float inv_dim = 1.f / float(D);
  // (the loop runs equally often in all lanes of a warp: its shuffles are whole-warp)
  for (int h0 = blockIdx.y * per_token; h0 < rows; h0 += step, head += step) {
    const bool live = active && head < rows;
    float x[2 * kUnit];
    next[0].widen(x), next[1].widen(x + kUnit);
    if (active && head + step < rows) next[0].load(source(head + step) + a), next[1].load(source(head + step) + b);  // in flight meanwhile
    if (norm) {
      float ss = 0.f;
      if (live) {
#pragma unroll
        for (int i = 0; i < 2 * kUnit; i++) ss = fmaf(x[i], x[i], ss);
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (live && head < qk_heads) {
        const float rms = rsqrtf(ss * inv_dim + p.eps);
        const float* w = weights + (head < p.q_heads ? 0 : D);
#pragma unroll
        for (int i = 0; i < kUnit; i += 4) {
          const float4 wa = *reinterpret_cast<const float4*>(w + a + i), wb = *reinterpret_cast<const float4*>(w + b + i);
          x[i] *= rms * wa.x, x[i + 1] *= rms * wa.y, x[i + 2] *= rms * wa.z, x[i + 3] *= rms * wa.w;
          x[kUnit + i] *= rms * wb.x, x[kUnit + i + 1] *= rms * wb.y, x[kUnit + i + 2] *= rms * wb.z, x[kUnit + i + 3] *= rms * wb.w;
        }
      }
    }
    if (!live) continue;
    if (head < qk_heads && turns) {
      if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < kUnit; i++) turn_pair(x[2 * i], x[2 * i + 1], cs[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kUnit; i++) turn_pair(x[i], x[i + kUnit], cs[i]);
      }
    }
    Out* dst;
    if (head < p.q_heads) {
      dst = static_cast<Out*>(p.q_out) + t * p.q_out_ld_token + head * p.q_out_ld_head;
    } else if (p.slots) {
      const int64_t place = place_of[tl];
      if (place < 0) continue;  // not written
      const int64_t page = place >> 32, at = place & 0xffffffff;
      dst = head < qk_heads ? static_cast<Out*>(p.k_cache) + page * p.kc_ld_page + (head - p.q_heads) * p.kc_ld_head + at * p.kc_ld_slot
                            : static_cast<Out*>(p.v_cache) + page * p.vc_ld_page + (head - qk_heads) * p.vc_ld_head + at * p.vc_ld_slot;
    } else {
      dst = static_cast<Out*>(p.k_out) + t * p.k_out_ld_token + (head - p.q_heads) * p.k_out_ld_head;
    }
    store<kUnit>(dst + a, x), store<kUnit>(dst + b, x + kUnit);
  }
}

size_t type_size(int dtype) { return dtype == Q27B_F32 ? 4 : 2; }

template <typename In, typename Out, int kUnit, int kLanes>
int launch(const Args& p, cudaStream_t s) {
  const int rows = p.q_heads + p.k_heads + (p.v ? p.k_heads : 0), groups = kThreads / kLanes;
  const int sms = sm_count();
  // Many tokens: four to a CTA, so that the cos / sin table costs about one evaluation per thread. Few: one to a CTA, and its
  // rows shared out over grid.y until the CTAs fill the GPU.
  const int tokens = p.T >= 4 * 4 * sms ? kMostTokens : 1;
  const int blocks = (p.T + tokens - 1) / tokens;
  int share = 1;
  while (tokens == 1 && blocks * share * 2 <= 2 * sms && share * groups < rows) share *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(blocks), unsigned(share)), cfg.blockDim = dim3(kThreads), cfg.stream = s;
  cfg.dynamicSmemBytes = size_t(tokens) * (p.rot_dim / 2) * sizeof(float2) + (p.q_weight ? 2 * size_t(p.head_dim) * sizeof(float) : 0);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 1 : 0;
  uint32_t* status = device_status_ptr();
  Q27B_REQUIRE(status, "qk_rope: no device status word");
  Q27B_CUDA(cudaLaunchKernelEx(&cfg, qk_rope_kernel<In, Out, kUnit, kLanes>, p, tokens, status));
  return 0;
}

// Whether a tensor can be loaded and stored `unit` channels at a time: base and strides in whole groups. Null passes.
bool grouped(int unit, const void* base, int dtype, int64_t ld0, int64_t ld1, int64_t ld2 = 0) {
  return reinterpret_cast<uintptr_t>(base) % std::min<size_t>(16, unit * type_size(dtype)) == 0 && ld0 % unit == 0 && ld1 % unit == 0 && ld2 % unit == 0;
}
bool all_grouped(int unit, const Args& p) {
  return grouped(unit, p.q, p.in_dtype, p.q_ld_token, p.q_ld_head) && grouped(unit, p.k, p.in_dtype, p.k_ld_token, p.k_ld_head) &&
         grouped(unit, p.v, p.in_dtype, p.v_ld_token, p.v_ld_head) && grouped(unit, p.q_out, p.out_dtype, p.q_out_ld_token, p.q_out_ld_head) &&
         grouped(unit, p.k_out, p.out_dtype, p.k_out_ld_token, p.k_out_ld_head) &&
         grouped(unit, p.k_cache, p.out_dtype, p.kc_ld_page, p.kc_ld_head, p.kc_ld_slot) &&
         grouped(unit, p.v_cache, p.out_dtype, p.vc_ld_page, p.vc_ld_head, p.vc_ld_slot);
}

// Sixteen channels to a lane where sizes and strides allow (half the index arithmetic per byte, 16-byte accesses of 16-bit
// types), else eight, with a whole warp to a row.
template <typename In, typename Out>
int launch_lanes(const Args& p, cudaStream_t s) {
  if (p.head_dim % 16 || p.rot_dim % 16 || !all_grouped(8, p)) return launch<In, Out, 4, 32>(p, s);
  if (p.head_dim <= 64) return launch<In, Out, 8, 4>(p, s);
  if (p.head_dim <= 128) return launch<In, Out, 8, 8>(p, s);
  return launch<In, Out, 8, 16>(p, s);
}

template <typename In>
int launch_out(const Args& p, cudaStream_t s) {
  if (p.out_dtype == Q27B_F32) return launch_lanes<In, float>(p, s);
  if (p.out_dtype == Q27B_BF16) return launch_lanes<In, __nv_bfloat16>(p, s);
  return launch_lanes<In, __half>(p, s);
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
  Q27B_REQUIRE(p.q && p.q_out && grouped(4, p.q, p.in_dtype, p.q_ld_token, p.q_ld_head) && grouped(4, p.q_out, p.out_dtype, p.q_out_ld_token, p.q_out_ld_head),
               "qk_norm_rope: q and q_out must not be null and must start and stride in whole groups of four channels");
  Q27B_REQUIRE(!p.q_weight == !p.k_weight || p.k_heads == 0, "qk_norm_rope: the norm needs both weights");
  if (p.q_weight) {
    const int wt = p.weight_f32 ? Q27B_F32 : Q27B_BF16;
    Q27B_REQUIRE(grouped(4, p.q_weight, wt, 0, 0) && (p.k_heads == 0 || grouped(4, p.k_weight, wt, 0, 0)), "qk_norm_rope: the weights must be aligned to four values");
    Q27B_REQUIRE(p.eps >= 0.f, "qk_norm_rope: eps must not be negative");
  }
  Q27B_REQUIRE(p.k_heads > 0 || (!p.k && !p.v && !p.slots), "qk_norm_rope: keys, values or slots without key heads");
  if (p.k_heads > 0) {
    Q27B_REQUIRE(p.k && grouped(4, p.k, p.in_dtype, p.k_ld_token, p.k_ld_head), "qk_norm_rope: k must not be null and must start and stride in whole groups of four channels");
    Q27B_REQUIRE(!p.v || (p.slots && grouped(4, p.v, p.in_dtype, p.v_ld_token, p.v_ld_head)),
                 "qk_norm_rope: v goes into the cache only, and must start and stride in whole groups of four channels");
    if (p.slots) {
      Q27B_REQUIRE(!p.k_out, "qk_norm_rope: keys go either to k_out or into the cache");
      Q27B_REQUIRE(p.page_size > 0 && p.pages > 0 && p.k_cache && grouped(4, p.k_cache, p.out_dtype, p.kc_ld_page, p.kc_ld_head, p.kc_ld_slot) &&
                       (!p.v || (p.v_cache && grouped(4, p.v_cache, p.out_dtype, p.vc_ld_page, p.vc_ld_head, p.vc_ld_slot))),
                   "qk_norm_rope: the cache must not be null or empty and must start and stride in whole groups of four channels");
    } else {
      Q27B_REQUIRE(p.k_out && grouped(4, p.k_out, p.out_dtype, p.k_out_ld_token, p.k_out_ld_head),
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
