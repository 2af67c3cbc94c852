// Prompts and chunks: many query rows per key head. Included by attention.cu.
//
// Work. The query rows of one key head (row = token x heads per key head: the heads of a group share their keys, so a tile of 128
// rows spans few positions and little of it is masked) are cut into segments of kTiles x 128 rows; a segment's work is
// its 128-key tiles, from the window and the sinks of its first row to the position of its last. As in the streaming kernel
// all segments' tiles are cut into equal ranges, one per SM, and the pieces of cut segments joined afterwards; a segment
// counts for kSegmentCost tiles more than it has (with 3 instead of 5 the CTA that gets a long prompt's first, short segments
// ends last and the kernel takes 8 % longer).
//
// Arithmetic, per 128-row tile: S = Q K^T by tcgen05.mma into tensor memory; two threads per row read half a row of S each, agree on
// the running maximum, write P = 2^(c s - c m) back over S in the inputs' type, and O += P V follows with P as the
// tensor-memory operand and V straight from its row-major tile (the transposed shared-memory operand form). O stays in tensor
// memory; it is scaled down only when a row's maximum has grown by more than 8 binary orders since the last time (P then
// stays below 2^8, exact to the same relative step), so that most tiles skip the round trip. P is rounded to the inputs' type for
// the second product, as the tensor cores take it; the sums add the unrounded values in fp32. Up to 128 channels two
// row tiles take turns: while one's softmax runs, the other's products do. At 256 channels O of one tile fills half the tensor
// memory; there is one row tile, with two S buffers, and S of the next tile is computed during the softmax.
//
// Roles: eight warps per row tile (softmax, scaling, epilogue, and the load of the next segment's Q), a warp per row tile that issues
// its products, two warps that issue the copies. K and V pass through one ring in the order in which the products use them.
//
// What bounds it: per pair of row tiles and 128 keys the products need 2048 cycles and the exponentials as many (a quarter less
// with those on the FMA units); measured are 3500. The rest is the chain from S over the softmax (1900 cycles, more than half of
// them exponentials and their conversions while both tiles compete for the same units) to P V and the next S (1100 and the signals
// between the warps). Measured on 8192 tokens, 40 heads over 8 of 128 channels, bf16, causal: 700 us, 980 TFLOP/s (60 % of the
// measured burst rate of a matrix product, 70 % of the sustained one; the power limit holds the clock at 1.5 to 1.7 GHz, and
// after seconds of load 800 us are measured); 512 tokens behind 24000 of 256 channels: 285 us, 1070 TFLOP/s. Tried and measured
// worse or equal: one thread per row (790 us against 766 at the time), 64-key tiles with two S buffers (1470 against 790: the cost
// per tile hardly depends on its size), both tiles' products issued by one warp in fixed order (820) or by two in strict turns
// (766 against 735), the two row tiles sharing a short segment's keys (no gain for verification).

template <int D>
struct TileCfg {
  static constexpr int kTiles = D == 256 ? 1 : 2;                // row tiles of a segment
  static constexpr int kRows = 128 * kTiles;
  static constexpr int kKeys = 128;
  // What a segment costs beside its tiles (Q, the start and the end of the pipeline, the epilogue), in tiles: it counts in the shares
  static constexpr int kSegmentCost = 5;
  // Whether pair x of a thread's exponentials goes through the FMA units: every fourth where two row tiles compete for the
  // special-function units (prompt of 8192: 733 -> 700 us; every third to sixth alike), none at 256 channels, where the products
  // take twice as long (chunk of 512: 285 us without, 301 with).
  static constexpr bool on_fma(int x) { return D != 256 && x % 4 == 1; }
  static constexpr int kParts = D == 256 ? 2 : 1;                // ring slots per K or V tile
  static constexpr int kSlotBytes = kKeys * D * 2 / kParts;
  static constexpr int kSlots = D == 64 ? 8 : 4;
  static constexpr int kQBytes = 128 * D * 2;
  static constexpr int kSoftmaxWarps = 8 * kTiles;
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 4);      // and a warpgroup for the products and the copies (two warps idle)
  // Two row tiles: 640 threads get 96 registers each at launch; the softmax takes 104, the others go down to 64:
  // 512 x 104 + 128 x 64 = 640 x 96, never more than the launch got.
  static constexpr int kLaunchRegs = 96, kSoftmaxRegs = 104, kOtherRegs = 64;
  static_assert(kTiles == 1 || 512 * kSoftmaxRegs + 128 * kOtherRegs <= 640 * kLaunchRegs, "registers");
  static constexpr int kSmemBytes = 1024 + kTiles * kQBytes + kSlots * kSlotBytes + 256;
  static constexpr int kPieceFloats = kRows * (D + 2);
  static constexpr int kO = 256;                                 // tensor-memory column of the (first) output; S at 0 and 128
};

__device__ __forceinline__ int tile_of(int i, int sink_tiles, int first_window_tile) { return i < sink_tiles ? i : first_window_tile + i - sink_tiles; }

// The key tiles that rows [row0, row1) of a sequence see (row = token x G).
struct TileRange {
  int low, reach;  // window start of the first row; keys [0, reach) can be seen by the last row
  int sink_tiles, first_window_tile, tiles;
  int pmin, pmax;
};
__device__ __forceinline__ TileRange tile_range(const Args& p, const Sequence& s, int G, int row0, int row1) {
  TileRange r;
  const int first = s.len - s.rows;
  r.pmin = first + row0 / G, r.pmax = first + (row1 - 1) / G;
  r.reach = max(min(r.pmax + 1, s.reach), 0);
  r.low = p.window > 0 ? max(r.pmin - p.window + 1, 0) : 0;
  r.sink_tiles = (min(min(p.sinks, r.low), r.reach) + 127) / 128;
  r.first_window_tile = max(r.low / 128, r.sink_tiles);
  r.tiles = max(r.sink_tiles + max((r.reach + 127) / 128 - r.first_window_tile, 0), 1);
  return r;
}

__device__ __forceinline__ int heavy_rows(const Args& p, const Sequence& s, int min_rows) {
  const int rows = s.rows * (p.heads / p.kv_heads);
  return rows >= min_rows ? rows : 0;
}

struct TileCursor {
  int b, hk, rt, from, rows;  // rows of the sequence; from: this CTA's first tile of the segment
  int64_t at;                 // where the segment's tiles begin in the order of all shares (its own cost lies before them)
  Sequence s;
  TileRange r;
  __device__ int end(int64_t t1) const { return int(max(int64_t(0), min(int64_t(r.tiles), t1 - at))); }  // of a range up to t1
  __device__ bool any(const Args& p, int64_t t1) const { return b < p.B && from < end(t1); }
  template <int kRows>
  __device__ void load(const Args& p) {
    r = tile_range(p, s, p.heads / p.kv_heads, rt * kRows, min((rt + 1) * kRows, rows));
  }
  template <int kRows, int kCost>
  __device__ void next(const Args& p, int min_rows) {
    from = 0, at += r.tiles + kCost;
    if (++rt * kRows >= rows) {
      rt = 0;
      if (++hk >= p.kv_heads) {
        hk = 0;
        do {
          if (++b >= p.B) return;
          s = sequence_of(p, b), rows = heavy_rows(p, s, min_rows);
        } while (rows == 0);
      }
    }
    load<kRows>(p);
  }
};

// Bits 0 .. n - 1.
__device__ __forceinline__ uint64_t below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

// The code of what seldom happens is laid out away from the loop, which is long enough to feel its instruction fetches.
__device__ __forceinline__ bool rarely(bool x) { return __builtin_expect(x, 0); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest, NaN if one is.
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// 2^x of two values on the FMA units (x <= 8; below -126 as -126): x = n + r with n the nearest integer, 2^r by a polynomial of
// degree 5 in r (fitted on [-1/2, 1/2] for the smallest relative error, 1 at 0: 2^-22 in fp32 arithmetic), n added to its exponent.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), unmagic = make_float2(-12582912.f, -12582912.f), minus = make_float2(-1.f, -1.f);
  x = make_float2(fmaxf(x.x, -126.f), fmaxf(x.y, -126.f));
  const float2 t = add2(x, magic);  // 1.5 2^23 + n: n in the low bits
  const float2 r = fma2(add2(t, unmagic), minus, x);
  float2 e = fma2(r, make_float2(1.326472731307149e-3f, 1.326472731307149e-3f), make_float2(9.671512991189957e-3f, 9.671512991189957e-3f));
  e = fma2(e, r, make_float2(5.550733581185341e-2f, 5.550733581185341e-2f));
  e = fma2(e, r, make_float2(0.24022242426872253f, 0.24022242426872253f));
  e = fma2(e, r, make_float2(0.6931470036506653f, 0.6931470036506653f));
  e = fma2(e, r, make_float2(1.f, 1.f));
  return make_float2(__int_as_float((__float_as_int(t.x) << 23) + __float_as_int(e.x)), __int_as_float((__float_as_int(t.y) << 23) + __float_as_int(e.y)));
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// D[tmem] (+)= A[smem] B[smem]^T and D[tmem] (+)= A[tmem] B[smem]; one thread issues.
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::f16: fp32 accumulator, both operands bf16 or both fp16, A K-major, 128 x n x 16.
__host__ __device__ constexpr uint32_t umma_idesc_f16(bool bf16, bool b_mn_major, uint32_t n) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// Shared-memory descriptor of an operand whose rows are K (keys) and whose 64-channel blocks of 128-byte rows carry the 128-byte
// swizzle: blocks `block_bytes` apart along N, groups of 8 keys 1024 bytes apart along K.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t block_bytes) {
  return uint64_t((smem_addr & 0x3FFFFu) >> 4) | (uint64_t(block_bytes >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

template <typename T2>
struct is_bf16 { static constexpr bool value = false; };
template <>
struct is_bf16<__nv_bfloat162> { static constexpr bool value = true; };

template <typename T2, int D>
__global__ void __launch_bounds__(TileCfg<D>::kThreads, 1)
    attention_tile_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                          const __grid_constant__ Args p, int min_rows, int box, float* pieces, JoinRecord* records, uint32_t* status) {
  using C = TileCfg<D>;
  constexpr int NT = C::kTiles;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t ring = base + NT * C::kQBytes;
  __shared__ uint64_t bars[2 * C::kSlots + 9];
  __shared__ volatile uint32_t abort_flag;
  __shared__ uint32_t tmem_word, issuing;
  __shared__ int64_t sums[20];
  // What the two threads of a row tell one another: maxima (by turns: a thread may be a tile ahead), sums.
  __shared__ float half_m[2][2][NT][128], half_l[2][NT][128];
  __shared__ int64_t start_off;
  __shared__ int start_b, start_rt, start_i;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  constexpr int kWarps = C::kThreads / 32;
  static_assert(kWarps <= 20, "sums");
  auto full = [&](int s) { return smem_u32(bars + s); };
  auto empty = [&](int s) { return smem_u32(bars + C::kSlots + s); };
  auto s_full = [&](int t) { return smem_u32(bars + 2 * C::kSlots + t); };
  auto p_ready = [&](int t) { return smem_u32(bars + 2 * C::kSlots + 2 + t); };
  auto q_ready = [&](int t) { return smem_u32(bars + 2 * C::kSlots + 4 + t); };
  auto pv_done = [&](int t) { return smem_u32(bars + 2 * C::kSlots + 6 + t); };
  const uint32_t drained = smem_u32(bars + 2 * C::kSlots + 8);

  if (tid == 0) {
    abort_flag = 0, issuing = 0, start_b = -1;
    for (int s = 0; s < C::kSlots; s++) mbar_init(full(s), 1), mbar_init(empty(s), NT);
    for (int t = 0; t < 2; t++) mbar_init(s_full(t), 1), mbar_init(p_ready(t), 8), mbar_init(q_ready(t), 8), mbar_init(pv_done(t), 1);
    mbar_init(drained, NT);
    mbar_init_fence();
    prefetch_tensormap(&kmap), prefetch_tensormap(&vmap);
  }
  pdl_wait();

  // ---- this CTA's range of the tiles: every warp sums a run of sequences, its lanes share a sequence's segments ---------------
  const int G = p.heads / p.kv_heads, run = (p.B + kWarps - 1) / kWarps, b_lo = min(warp * run, p.B), b_hi = min(b_lo + run, p.B);
  auto cost_of = [&](const Sequence& s, int rows) {  // of all segments of one key head, over the lanes
    int n = 0;
    for (int rt = lane; rt * C::kRows < rows; rt += 32) n += C::kSegmentCost + tile_range(p, s, G, rt * C::kRows, min((rt + 1) * C::kRows, rows)).tiles;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
  };
  auto each_heavy = [&](auto&& f) {  // f(b, sequence, rows) for the warp's sequences that this kernel takes
    for (int b0 = b_lo; b0 < b_hi; b0 += 32) {
      const int b = b0 + lane;
      Sequence s = {};
      int rows = 0;
      if (b < b_hi) s = sequence_of(p, b), rows = heavy_rows(p, s, min_rows);
      for (uint32_t left = __ballot_sync(0xffffffffu, rows > 0); left; left &= left - 1) {
        const int from = __ffs(left) - 1;
        Sequence u;
        u.row0 = __shfl_sync(0xffffffffu, s.row0, from), u.rows = __shfl_sync(0xffffffffu, s.rows, from);
        u.len = __shfl_sync(0xffffffffu, s.len, from), u.reach = __shfl_sync(0xffffffffu, s.reach, from);
        f(b0 + from, u, __shfl_sync(0xffffffffu, rows, from));
      }
    }
  };
  int64_t mine = 0;
  each_heavy([&](int, const Sequence& s, int rows) { mine += int64_t(p.kv_heads) * cost_of(s, rows); });
  if (lane == 0) sums[warp] = mine;
  __syncthreads();
  int64_t total = 0, before = 0;
  for (int w = 0; w < kWarps; w++) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  const int64_t ctas = min(int64_t(gridDim.x), total), c = blockIdx.x;
  if (c >= ctas) {
    if (tid == 0) records[c].pieces = 0;
    return;
  }
  const int64_t t0 = total * c / ctas, t1 = total * (c + 1) / ctas;
  if (before <= t0 && t0 < before + mine) {
    each_heavy([&](int b, const Sequence& s, int rows) {
      const int n = cost_of(s, rows);
      const int64_t w = int64_t(p.kv_heads) * n;
      if (before <= t0 && t0 < before + w) {
        int off = int((t0 - before) % n);  // among one key head's segments
        int acc = 0;
        for (int r0 = 0; r0 * C::kRows < rows; r0 += 32) {
          const int rt = r0 + lane;
          const int m = rt * C::kRows < rows ? C::kSegmentCost + tile_range(p, s, G, rt * C::kRows, min((rt + 1) * C::kRows, rows)).tiles : 0;
          int upto = m;
#pragma unroll
          for (int o = 1; o < 32; o *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
          }
          if (m > 0 && acc + upto - m <= off && off < acc + upto) start_b = b, start_off = (t0 - before) / n, start_rt = rt, start_i = off - (acc + upto - m);
          acc += __shfl_sync(0xffffffffu, upto, 31);
        }
      }
      before += w;
    });
  }
  if (warp == 0) {  // (after the exit above: what is taken is given back)
    tmem_alloc(smem_u32(&tmem_word), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // Only now: a successor that starts early beside this CTA and takes tensor memory of its own before it waits for this kernel
  // would hold what this CTA still had to take.
  pdl_trigger();
  const uint32_t tmem = tmem_word;
  TileCursor cur;
  cur.b = start_b;
  const bool work = cur.b >= 0;  // (false: the lengths changed under the kernel)
  if (work) {
    cur.s = sequence_of(p, cur.b), cur.rows = heavy_rows(p, cur.s, min_rows);
    cur.hk = int(start_off), cur.rt = start_rt;
    cur.template load<C::kRows>(p);
    // (start_i: the position within the segment, its own cost first)
    cur.from = max(start_i - C::kSegmentCost, 0), cur.at = t0 - start_i + C::kSegmentCost;
  }
  if (tid == 0) {
    JoinRecord r = {0, cur.b, cur.hk, cur.rt};
    if (work) {
      const int64_t s1 = cur.at + cur.r.tiles;
      if (cur.from > 0 && total * (c - 1) / ctas <= cur.at) r.pieces = int((s1 * ctas + total - 1) / total - 1 - c) + 2;
    }
    records[c] = r;
  }

  if (warp >= C::kSoftmaxWarps) {
    if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
  // (the other warps are idle: they complete the warpgroup)
  if (warp == C::kSoftmaxWarps + NT || warp == C::kSoftmaxWarps + NT + 1) {
    // ---- copies: two warps issue every other ring slot each (one would spend longer on it than the products take) --------------
    const int turn_of = warp - C::kSoftmaxWarps - NT;
    const int boxes = C::kKeys / box, page_bits = __ffs(p.page_size) - 1;  // boxes per tile: at most eight, one per lane
    int slot = 0, issued = 0;
    uint32_t phase = 0;
    bool stop = false;  // a wait ran out (the same in all lanes)
    // Lane x looks after box x of a tile: where it lies, and whether a row sees any of its page (others are not read).
    struct Box {
      int tile0, k0, page;
      bool need;
    };
    auto look_up = [&](int i) {
      Box x;
      x.tile0 = tile_of(i, cur.r.sink_tiles, cur.r.first_window_tile) * C::kKeys;
      x.k0 = x.tile0 + lane * box, x.page = 0;
      const int k1 = min(x.k0 + box, cur.r.reach);
      x.need = lane < boxes && x.k0 < cur.r.reach && (x.k0 < p.sinks || k1 > cur.r.low);
      if (x.need) x.page = p.table[cur.b * p.table_ld + (x.k0 >> page_bits)];
      return x;
    };
    auto load = [&](const CUtensorMap* map, bool values, const Box& x) {  // all lanes
      if (stop) return;
      const int tile0 = x.tile0;
      int page = x.page;
      if (x.need && (page < 0 || page >= p.pages)) page = p.pages, atomicCAS(status, 0u, uint32_t(kStatusBadPage));  // (reads zeros)
      const uint32_t needs = __ballot_sync(0xffffffffu, x.need);
#pragma unroll
      for (int part = 0; part < C::kParts; part++) {
        // K is split along its channels, V along its keys
        const uint32_t in_part = C::kParts == 1 || !values ? needs : needs & (((1u << (boxes / 2)) - 1u) << (part * (boxes / 2)));
        constexpr int kBlocks = D / 64;
        const int d0 = C::kParts == 2 && !values ? part * kBlocks / 2 : 0, dn = C::kParts == 2 && !values ? kBlocks / 2 : kBlocks;
        const int rows = C::kParts == 2 && values ? C::kKeys / 2 : C::kKeys;
        if ((issued & 1) != turn_of) {  // the other warp's
          issued++;
          if (++slot == C::kSlots) slot = 0, phase ^= 1u;
          continue;
        }
        if (issued >= C::kSlots && !warp_wait(empty(slot), phase ^ 1u, &abort_flag, status, kStatusEmptyWaitTimeout, 0)) {
          stop = true;
          return;
        }
        // One elected lane issues, with the boxes' pages from the lanes that looked them up: copies issued by several lanes of a
        // warp go out one lane at a time, at 190 cycles each.
        const uint32_t dst = ring + slot * C::kSlotBytes, bar = full(slot);
        if (elect_one()) mbar_arrive_expect_tx(bar, uint32_t(__popc(in_part) * dn * box) * 128u);
        for (uint32_t left = in_part; left; left &= left - 1) {
          const int lane_of = __ffs(left) - 1, page_of = __shfl_sync(0xffffffffu, page, lane_of);
          const int at = tile0 + lane_of * box, in_tile = lane_of * box - (rows < C::kKeys ? part * rows : 0);
          if (elect_one()) {
#pragma unroll
            for (int d = 0; d < kBlocks; d++)
              if (d < dn) tma_load_4d(dst + (d * rows + in_tile) * 128, map, (d0 + d) * 64, at & (p.page_size - 1), cur.hk, page_of, bar);
          }
          __syncwarp();
        }
        issued++;
        if (++slot == C::kSlots) slot = 0, phase ^= 1u;
      }
    };
    if (work)
      for (; cur.any(p, t1) && !stop; cur.template next<C::kRows, C::kSegmentCost>(p, min_rows)) {
        const int from = cur.from, end = cur.end(t1);
        if (cur.s.len > cur.s.reach && lane == 0) atomicCAS(status, 0u, uint32_t(kStatusBadPage));
        // In the order in which the products use them. The table is read a tile ahead: its latency would add to the copy's.
        Box x = look_up(from);
        load(&kmap, false, x);
        for (int i = from; i < end; i++) {
          const Box next = i + 1 < end ? look_up(i + 1) : x;
          if (NT == 1 && i + 1 < end) load(&kmap, false, next);
          load(&vmap, true, x);
          if (NT == 2 && i + 1 < end) load(&kmap, false, next);
          x = next;
        }
      }
    if (stop)  // unwinding: no copy may still be in flight when the CTA ends
      for (int s = 0; s < C::kSlots && s < issued; s++) {
        if ((s & 1) != turn_of) continue;  // (the number of slots is even)
        const int last = issued - 1 - ((issued - 1 - s) % C::kSlots + C::kSlots) % C::kSlots;  // last use of slot s
        uint32_t unused = 0;
        if (lane == 0) mbar_wait_bounded(full(s), uint32_t(last / C::kSlots) & 1u, &abort_flag, &unused, kStatusDrainTimeout);
      }
  } else if (warp < C::kSoftmaxWarps + NT) {
    // ---- products -----------------------------------------------------------------------------------------------------------
    // The whole warp walks the segments and waits, so that addresses and descriptors stay uniform; one elected lane issues. (A
    // single-lane branch spent 115 cycles per product on moving descriptors, more than the products take.)
    if (work) {
      constexpr uint32_t qk_idesc = umma_idesc_f16(is_bf16<T2>::value, false, C::kKeys), pv_idesc = umma_idesc_f16(is_bf16<T2>::value, true, D);
      constexpr int kPartKeys = C::kKeys / C::kParts;
      const uint64_t q_desc = umma_desc_k_sw128(base), k_desc = umma_desc_k_sw128(ring), v_desc = umma_desc_mn_sw128(ring, kPartKeys * 128);
      int slot = 0;
      uint32_t phase = 0, p_phase = 0, q_phase = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity, uint32_t code) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(bar, parity, &abort_flag, status, code));
        tc_fence_after_sync();
      };
      auto advance = [&] { if (++slot == C::kSlots) slot = 0, phase ^= 1u; };
      // S of row tile t into buffer `buf` from the K part in ring slot s
      auto qk_part = [&](int t, int buf, int s, int part) {
        const uint64_t qd = q_desc + uint64_t((t * C::kQBytes + part * (C::kQBytes / C::kParts)) >> 4), kd = k_desc + uint64_t(s * (C::kSlotBytes >> 4));
        const uint32_t d = tmem + buf * 128;
#pragma unroll
        for (int k = 0; k < D / 16 / C::kParts; k++) {
          const uint32_t off = ((k / 4) * C::kKeys * 128 + (k % 4) * 32) >> 4;  // (the rows of Q's blocks are as many as K's)
          umma_f16_ss(d, qd + off, kd + off, qk_idesc, part + k > 0);
        }
      };
      auto pv_part = [&](int t, int buf, int s, int part, bool accumulate) {
        const uint64_t vd = v_desc + uint64_t(s * (C::kSlotBytes >> 4));
        const uint32_t d = tmem + C::kO + t * D, a = tmem + buf * 128 + part * 64;
#pragma unroll
        for (int k = 0; k < kPartKeys / 16; k++) umma_f16_ts(d, a + (k / 4) * 64 + (k % 4) * 8, vd + ((k * 2048) >> 4), pv_idesc, k > 0 || accumulate);
      };
      const int mine = warp - C::kSoftmaxWarps;
      for (; cur.any(p, t1) && ok; cur.template next<C::kRows, C::kSegmentCost>(p, min_rows)) {
        const int from = cur.from, end = cur.end(t1);
        if constexpr (NT == 2) {
          // A warp per row tile: while one waits, the other's products keep the tensor cores busy. They do not issue at the same time:
          // products of both tiles mixed together would end together, and so would the softmaxes between them. (The lock orders work and
          // guards nothing: a warp that does not get it in time goes on without.) A tile without rows in this segment only gives the
          // ring slots back.
          const bool both = cur.rows - cur.rt * C::kRows > 128;
          auto lock = [&] {
            for (int i = 0; both && i < 4096 && atomicCAS(&issuing, 0u, 1u) != 0u; i++) {}
          };
          auto unlock = [&] {
            if (both) atomicExch(&issuing, 0u);
          };
          if (both || mine == 0) {
            wait(q_ready(mine), q_phase, kStatusAccumWaitTimeout), q_phase ^= 1u;
            wait(full(slot), phase, kStatusFullWaitTimeout);
            if (!ok) break;
            if (elect_one()) lock(), qk_part(mine, mine, slot, 0), umma_commit(s_full(mine)), unlock(), umma_commit(empty(slot));
            __syncwarp();
            advance();
            for (int i = from; i < end; i++) {
              const int vs = slot;
              wait(full(slot), phase, kStatusFullWaitTimeout);  // V of this tile
              advance();
              const bool more = i + 1 < end;
              if (more) wait(full(slot), phase, kStatusFullWaitTimeout);  // K of the next
              wait(p_ready(mine), p_phase, kStatusAccumWaitTimeout), p_phase ^= 1u;
              if (!ok) break;
              if (elect_one()) {
                lock();
                pv_part(mine, mine, vs, 0, i > from);
                if (more)
                  qk_part(mine, mine, slot, 0), umma_commit(s_full(mine)), unlock(), umma_commit(empty(vs)), umma_commit(empty(slot));
                else
                  umma_commit(pv_done(mine)), unlock(), umma_commit(empty(vs));
              }
              __syncwarp();
              if (more) advance();
            }
          } else {
            for (int i = 0; i < 2 * (end - from) && ok; i++) {
              wait(full(slot), phase, kStatusFullWaitTimeout);
              if (lane == 0) mbar_arrive(empty(slot));
              advance();
            }
          }
        } else {
          auto qk = [&](int buf) {
            for (int part = 0; part < C::kParts && ok; part++) {
              wait(full(slot), phase, kStatusFullWaitTimeout);
              if (ok && elect_one()) {
                qk_part(0, buf, slot, part);
                umma_commit(empty(slot));
                if (part == C::kParts - 1) umma_commit(s_full(buf));
              }
              __syncwarp();
              advance();
            }
          };
          wait(q_ready(0), q_phase, kStatusAccumWaitTimeout), q_phase ^= 1u;
          int buf = 0;  // of the tile whose P comes next; every segment starts at 0
          qk(0);
          for (int i = from; i < end && ok; i++) {
            if (i + 1 < end) qk(buf ^ 1);
            wait(p_ready(buf), (p_phase >> buf) & 1u, kStatusAccumWaitTimeout), p_phase ^= 1u << buf;  // (bit b: of S buffer b)
            for (int part = 0; part < C::kParts && ok; part++) {
              wait(full(slot), phase, kStatusFullWaitTimeout);
              if (ok && elect_one()) {
                pv_part(0, buf, slot, part, part > 0 || i > from);
                umma_commit(empty(slot));
                if (part == C::kParts - 1) umma_commit(pv_done(0));
              }
              __syncwarp();
              advance();
            }
            buf ^= 1;
          }
        }
      }
      if (elect_one()) umma_commit(drained);  // no product may be in flight when the tensor memory is given back, after a failed wait either
      __syncwarp();
      uint32_t unused = 0;
      mbar_wait_bounded(drained, 0, &unused, nullptr, kStatusDrainTimeout);
    }
    __syncwarp();
  }
  } else {
    if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    // ---- softmax, scaling, epilogue: two threads per row, each with half the keys of S and half the channels of O ------------------
    const int tile = warp / 8, half = (warp / 4) % 2, row_in_tile = (warp % 4) * 32 + lane;
    const uint32_t lanes = uint32_t(32 * (warp % 4)) << 16, o_at = tmem + lanes + C::kO + tile * D + half * (D / 2);
    const float c2 = p.scale * 1.4426950408889634f, scale_log2 = c2 > 0.f ? c2 : 1e-30f;  // (0 would turn a masked -infinity into NaN)
    auto pair_bar = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + tile * 4 + warp % 4) : "memory"); };  // the two warps of 32 rows
    uint32_t s_phase = 0, pv_phase = 0;  // (bit b: of S buffer b)
    int chunk = 0;  // ring places used before this segment
    // This thread's half of its row of the segment at `at` starts on its way into shared memory, in the layout of the products'
    // operands (zeros for a row that is not there); q_here hands it over.
    auto load_q = [&](const TileCursor& at) {
      const int row = at.rt * C::kRows + tile * 128 + row_in_tile;
      const bool live = row < at.rows;
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + (live ? (at.s.row0 + row / G) * p.q_ld_token + (at.hk * G + row % G) * p.q_ld_head : 0);
      const uint32_t dst = base + tile * C::kQBytes + row_in_tile * 128;
#pragma unroll
      for (int x = 0; x < D / 16; x++) {
        const int d = half * (D / 16) + x;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (d / 8) * 128 * 128 + (((d % 8) ^ (row_in_tile & 7)) << 4)), "l"(src + d * 8), "r"(live ? 16 : 0) : "memory");
      }
    };
    auto q_here = [&] {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready(tile));
    };
    auto in_use = [&](const TileCursor& at) { return at.rows - at.rt * C::kRows > tile * 128; };
    if (work && cur.any(p, t1) && in_use(cur)) load_q(cur), q_here();
    while (work && cur.any(p, t1)) {
      const int from = cur.from, end = cur.end(t1);
      auto load_next_q = [&](TileCursor nxt) {
        nxt.template next<C::kRows, C::kSegmentCost>(p, min_rows);
        const bool any = nxt.any(p, t1) && in_use(nxt);
        if (any) load_q(nxt);
        return any;
      };
      bool next_q = false;  // the next segment's Q is on its way
      if (in_use(cur)) {
        const int row = cur.rt * C::kRows + tile * 128 + row_in_tile, row_end = min(cur.rows, cur.rt * C::kRows + tile * 128 + 128);
        const int first = cur.s.len - cur.s.rows, pos = first + row / G;
        const bool warp_live = cur.rt * C::kRows + tile * 128 + (warp % 4) * 32 < cur.rows;  // a warp without rows only keeps step
        // Tiles that start in [whole_lo, whole_hi) or before whole_sinks are seen in full by every row of this row tile; those in
        // [held_lo, held_hi) or before held_sinks hold no key that no row of the segment sees.
        const int pmin = first + (cur.rt * C::kRows + tile * 128) / G, pmax = first + (row_end - 1) / G;
        const int whole_hi = min(pmin + 1, cur.r.reach) - C::kKeys + 1, whole_lo = p.window > 0 ? pmax - p.window + 1 : 0;
        const int held_hi = cur.r.reach - C::kKeys + 1, held_lo = cur.r.low, sinks_hi = p.sinks - C::kKeys + 1;
        float m = -INFINITY, l = 0.f, mc = 0.f;  // mc: what is taken off the scaled scores
        for (int i = from; i < end; i++) {
          const int buf = NT == 2 ? tile : (i - from) & 1;
          const uint32_t s_at = tmem + lanes + buf * 128 + half * 64;
          const int k0 = tile_of(i, cur.r.sink_tiles, cur.r.first_window_tile) * C::kKeys;
          const bool edge = !(k0 < whole_hi && (k0 >= whole_lo || k0 < sinks_hi));
          const bool here = mbar_wait_bounded(s_full(buf), (s_phase >> buf) & 1u, &abort_flag, status, kStatusAccumWaitTimeout);
          s_phase ^= 1u << buf;
          tc_fence_after_sync();
          // every product with this segment's Q has ended: the next segment's takes its place while the last softmax runs
          if (rarely(i == end - 1)) next_q = load_next_q(cur);
          auto wait_pv = [&] {  // of the tile before (kTiles == 1): it may still be adding to O
            mbar_wait_bounded(pv_done(0), pv_phase ^ 1u, &abort_flag, status, kStatusAccumWaitTimeout);
            tc_fence_after_sync();
          };
          if (warp_live) {
            // The maximum needs all 64 scores, the exponentials 32 at a time: they are read from tensor memory twice instead of being held.
            float tile_m;
            {
              float s[64];
              tmem_ld32(s_at, s), tmem_ld32(s_at + 32, s + 32);
              tmem_ld_wait();
              if (rarely(edge)) {
                // bit x: this row sees key at + x
                const int at = k0 + half * 64, hi = min(pos, cur.r.reach - 1) - at, lo = p.window > 0 ? pos - p.window + 1 - at : 0, si = p.sinks - at;
                const uint64_t seen = below(hi + 1) & (~below(lo) | below(si));
                const uint32_t seen0 = uint32_t(seen), seen1 = uint32_t(seen >> 32);
#pragma unroll
                for (int x = 0; x < 32; x++) s[x] = (seen0 >> x) & 1u ? s[x] : -INFINITY, s[x + 32] = (seen1 >> x) & 1u ? s[x + 32] : -INFINITY;
                tmem_st32(s_at, reinterpret_cast<uint32_t*>(s)), tmem_st32(s_at + 32, reinterpret_cast<uint32_t*>(s + 32));
                tmem_st_wait();
              }
              float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
              for (int x = 4; x < 60; x += 2) top[(x / 2) & 3] = max3(top[(x / 2) & 3], s[x], s[x + 1]);
              top[0] = max3(top[0], s[60], s[61]), top[1] = max3(top[1], s[62], s[63]);
              tile_m = max2(max3(top[0], top[1], top[2]), top[3]);
            }
            half_m[(i - from) & 1][half][tile][row_in_tile] = tile_m;
            pair_bar();
            tile_m = max2(tile_m, half_m[(i - from) & 1][half ^ 1][tile][row_in_tile]);
            // (m = -infinity: everything that is seen grows; a NaN is taken over and makes the row NaN)
            const bool grow = !((tile_m - m) * scale_log2 <= 8.f) && tile_m != -INFINITY;
            if (rarely(__any_sync(0xffffffffu, grow))) {
              const float f = grow ? exp2_fast((m - tile_m) * scale_log2) : 1.f;  // (m = -infinity: 0)
              if (grow) m = tile_m, mc = m * scale_log2, l *= f;
              if (mc == INFINITY) mc = NAN;  // an infinite score: infinity - infinity, for the polynomial's pairs too
              if (i > from) {
                if (NT == 1) wait_pv();
#pragma unroll
                for (int d = 0; d < D / 2; d += 32) {
                  float o[32];
                  tmem_ld32(o_at + d, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int x = 0; x < 32; x++) o[x] *= f;
                  tmem_st32(o_at + d, reinterpret_cast<uint32_t*>(o));
                }
              }
            }
            const float2 scale2 = make_float2(scale_log2, scale_log2), off2 = make_float2(-mc, -mc);
            float2 sum[2] = {};
#pragma unroll
            for (int h = 0; h < 2; h++) {
              float s[32];
              uint32_t w[16];
              tmem_ld32(s_at + 32 * h, s);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 16; x++) {
                float2 e = fma2(make_float2(s[2 * x], s[2 * x + 1]), scale2, off2);
                // the special-function units alone would need as long as the products: some of the pairs go through the FMA units
                e = C::on_fma(x) ? exp2_poly(e) : make_float2(exp2_fast(e.x), exp2_fast(e.y));
                sum[x & 1] = add2(sum[x & 1], e);
                T2 v;
                narrow(e, &v);
                w[x] = *reinterpret_cast<uint32_t*>(&v);
              }
              tmem_st16(s_at + 16 * h, reinterpret_cast<const uint4(&)[4]>(w));  // (over scores that have been read)
            }
            sum[0] = add2(sum[0], sum[1]);
            l += sum[0].x + sum[0].y;
            tmem_st_wait();
          }
          if (NT == 1) {
            // The product of the tile before is awaited in every turn, whether O was scaled or not: were it left running, its phase and
            // that of this tile's product could not be told apart.
            if (i > from) wait_pv();
            pv_phase ^= 1u;
          }
          // Values of keys that no row of the segment sees are whatever the cache (or an earlier tile) left there, and 0 x NaN would be
          // NaN: each row tile clears them before its own product, two threads to a key.
          if (rarely(edge && here && !(k0 < held_hi && (k0 >= held_lo || k0 < sinks_hi)))) {
            const int key = k0 + row_in_tile;
            const bool any = key < cur.r.reach && (key >= held_lo || key < p.sinks);
            const int n = end - from, j = i - from;
            int at = chunk + (NT == 2 ? 2 * j + 1 : C::kParts * min(2 * j + 2, 2 * n - 1));  // ring place of this V tile
            constexpr int kPartKeys = C::kKeys / C::kParts;
            at += row_in_tile / kPartKeys;
            if (!any) {
              mbar_wait_bounded(full(at % C::kSlots), uint32_t(at / C::kSlots) & 1u, &abort_flag, status, kStatusFullWaitTimeout);
              const uint32_t dst = ring + (at % C::kSlots) * C::kSlotBytes + (row_in_tile % kPartKeys) * 128 + half * 64;
#pragma unroll
              for (int d = 0; d < D / 64; d++)
#pragma unroll
                for (int x = 0; x < 4; x++)
                  asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(dst + d * kPartKeys * 128 + x * 16), "r"(0) : "memory");
              fence_proxy_async_smem();
            }
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_ready(buf));
        }
        if (next_q) q_here();
        // the last product of the segment, then its result
        const bool done = mbar_wait_bounded(pv_done(tile), NT == 2 ? pv_phase : pv_phase ^ 1u, &abort_flag, status, kStatusAccumWaitTimeout);
        if (NT == 2) pv_phase ^= 1u;
        if (warp_live) {
          tc_fence_after_sync();
          half_l[half][tile][row_in_tile] = l;
          pair_bar();
          l += half_l[half ^ 1][tile][row_in_tile];
          if (m == -INFINITY) l = 0.f;  // (a row that sees nothing: the polynomial's 2^-126s are no sum)
          const bool whole = from == 0 && end == cur.r.tiles, live = row < cur.rows && done;
          const float inv = l == 0.f ? 0.f : 1.f / l;
          uint16_t* out = static_cast<uint16_t*>(p.out) + (cur.s.row0 + row / G) * p.out_ld_token + (cur.hk * G + row % G) * p.out_ld_head + half * (D / 2);
          float* piece = pieces + (2 * c + (from > 0 ? 0 : 1)) * C::kPieceFloats;
#pragma unroll
          for (int d = 0; d < D / 2; d += 32) {
            float o[32];
            tmem_ld32(o_at + d, o);
            tmem_ld_wait();
            if (whole && live) {
#pragma unroll
              for (int x = 0; x < 32; x += 8) {
                T2 w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) narrow(l == 0.f ? make_float2(0.f, 0.f) : make_float2(o[x + 2 * e] * inv, o[x + 2 * e + 1] * inv), &w[e]);
                *reinterpret_cast<uint4*>(out + d + x) = *reinterpret_cast<uint4*>(w);
              }
            }
            if (!whole && live) {  // channel groups of four, rows side by side: a warp's stores are contiguous
#pragma unroll
              for (int x = 0; x < 32; x += 4)
                *reinterpret_cast<float4*>(piece + ((half * (D / 2) + d + x) / 4 * C::kRows + tile * 128 + row_in_tile) * 4) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
            }
          }
          if (half == 0) {
            const float mb = m * scale_log2;  // (-infinity stays)
            if (whole && live && p.lse) p.lse[int64_t(cur.s.row0 + row / G) * p.heads + cur.hk * G + row % G] = l == 0.f ? -INFINITY : (mb + log2f(l)) * 0.6931471805599453f;
            if (!whole && live) piece[C::kRows * D + tile * 128 + row_in_tile] = mb, piece[C::kRows * (D + 1) + tile * 128 + row_in_tile] = l;
          }
          tc_fence_before_sync();
        }
      } else if (load_next_q(cur)) {
        q_here();
      }
      chunk += 2 * (end - from) * C::kParts;
      cur.template next<C::kRows, C::kSegmentCost>(p, min_rows);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// Joins the pieces of the cut segments: block (c, y, z) takes 128 rows and 32 channels of the segment whose first cut is the
// start of CTA c's range.
template <typename T2, int D>
__global__ void __launch_bounds__(128) attention_tile_join_kernel(const __grid_constant__ Args p, const float* pieces, const JoinRecord* records) {
  using C = TileCfg<D>;
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x, in_seg = blockIdx.y * 128 + threadIdx.x, d0 = blockIdx.z * 32;
  const JoinRecord r = records[c];
  if (r.pieces == 0) return;
  const Sequence s = sequence_of(p, r.b);
  const int G = p.heads / p.kv_heads, row = r.rg * C::kRows + in_seg;
  if (row >= s.rows * G) return;
  auto piece = [&](int i) { return pieces + int64_t(i == 0 ? 2 * (c - 1) + 1 : 2 * (c - 1 + i)) * C::kPieceFloats; };
  float m = -INFINITY, l = 0.f;
  for (int i = 0; i < r.pieces; i++) m = fmaxf(m, piece(i)[C::kRows * D + in_seg]);
  float4 o[8] = {};
  for (int i = 0; i < r.pieces; i++) {
    const float* x = piece(i);
    const float mi = x[C::kRows * D + in_seg], f = exp2_fast(mi - m);
    if (mi == -INFINITY) continue;
    l += f * x[C::kRows * (D + 1) + in_seg];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float4 v = *reinterpret_cast<const float4*>(x + ((d0 / 4 + e) * C::kRows + in_seg) * 4);
      o[e].x += f * v.x, o[e].y += f * v.y, o[e].z += f * v.z, o[e].w += f * v.w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = static_cast<uint16_t*>(p.out) + (s.row0 + row / G) * p.out_ld_token + (r.hk * G + row % G) * p.out_ld_head + d0;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    T2 w[4];
    narrow(make_float2(o[e].x * inv, o[e].y * inv), &w[0]), narrow(make_float2(o[e].z * inv, o[e].w * inv), &w[1]);
    narrow(make_float2(o[e + 1].x * inv, o[e + 1].y * inv), &w[2]), narrow(make_float2(o[e + 1].z * inv, o[e + 1].w * inv), &w[3]);
    *reinterpret_cast<uint4*>(out + 4 * e) = *reinterpret_cast<uint4*>(w);
  }
  if (p.lse && blockIdx.z == 0) p.lse[int64_t(s.row0 + row / G) * p.heads + r.hk * G + row % G] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <int D>
size_t tile_scratch_bytes(int ctas) {
  return (size_t(ctas) * sizeof(JoinRecord) + 255) / 256 * 256 + size_t(ctas) * 2 * TileCfg<D>::kPieceFloats * 4;
}

template <typename T2, int D>
int launch_tile(const Args& p, int min_rows, void* ws, cudaStream_t s, uint32_t* status) {
  using C = TileCfg<D>;
  auto kernel = attention_tile_kernel<T2, D>;
  static bool done[64] = {};
  int dev = 0;
  Q27B_CUDA(cudaGetDevice(&dev));
  if (!(dev < 64 && done[dev])) {
    Q27B_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    if (C::kTiles == 2) {  // (a build that gave the launch fewer registers than the warpgroups then ask for would wait for them for ever)
      cudaFuncAttributes attrs;
      Q27B_CUDA(cudaFuncGetAttributes(&attrs, kernel));
      Q27B_REQUIRE(attrs.numRegs >= C::kLaunchRegs, "attention: the kernel was built with %d registers instead of %d", attrs.numRegs, C::kLaunchRegs);
    }
    if (dev < 64) done[dev] = true;
  }
  CUtensorMap km, vm;
  const int box = std::min(p.page_size, C::kKeys / C::kParts);
  if (int rc = make_cache_map(&km, p, p.k_cache, p.kc_ld_page, p.kc_ld_head, p.kc_ld_slot, box)) return rc;
  if (int rc = make_cache_map(&vm, p, p.v_cache, p.vc_ld_page, p.vc_ld_head, p.vc_ld_slot, box)) return rc;
  const int ctas = sm_count();
  JoinRecord* records = static_cast<JoinRecord*>(ws);
  float* pieces = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + (size_t(ctas) * sizeof(JoinRecord) + 255) / 256 * 256);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas)), cfg.blockDim = dim3(C::kThreads), cfg.dynamicSmemBytes = C::kSmemBytes, cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 1 : 0;
  Q27B_CUDA(cudaLaunchKernelEx(&cfg, kernel, km, vm, p, min_rows, box, pieces, records, status));
  cfg.gridDim = dim3(unsigned(ctas), C::kTiles, D / 32), cfg.blockDim = dim3(128), cfg.dynamicSmemBytes = 0;
  Q27B_CUDA(cudaLaunchKernelEx(&cfg, attention_tile_join_kernel<T2, D>, p, static_cast<const float*>(pieces), static_cast<const JoinRecord*>(records)));
  return 0;
}
