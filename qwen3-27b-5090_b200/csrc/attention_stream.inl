// The weight of a decode step outside the projections: few query rows per key head, so the keys and values are read once from
// HBM and that is the bound. Included by attention.cu. Measured: 16 sequences of 20000 to 32767 tokens, 8 key heads of 128
// channels in pages of 16: 261 us, 6.6 TB/s (101 % of the measured copy rate; 64 % when a single lane issued all copies);
// 64 sequences with a window of 4096: 168 us, 6.1 TB/s; one sequence of 131072 tokens: 91 us, 5.9 TB/s; one of 700: 11 us,
// the latency of two launches.
//
// Work. A segment is (sequence, key head, group of 16 query rows); its work is the 64-key tiles that its sequence sees. All
// segments' tiles, in order, are cut into equal ranges, one per resident CTA, whatever the lengths: no CTA waits for the
// longest sequence. A CTA finishes the segments that lie inside its range; of the at most two that its range cuts it leaves
// (running maximum, sum, unnormalised output) in the scratch, and a second small kernel joins the pieces in range order, so
// that the result does not depend on timing. The cuts depend on the lengths, which the kernel reads on the device: a captured
// launch follows them.
//
// Arithmetic. One producer warp keeps a ring of K / V tiles full by TMA, a box per page and 64 channels (128-byte swizzle).
// Four warps take 16 keys of each tile: S = Q K^T on mma.sync with the query rows (row = token x heads per key head) as the
// 16-row operand, the softmax in registers (the accumulator's layout is the next product's operand layout), O += P V. Each
// warp keeps its own maximum and sum; they meet at the end of the segment. mma.sync, not tcgen05: 16 rows would leave
// seven eighths of a 128-row tensor-memory tile idle, the round trip through tensor memory costs more than the products, and at
// 16 rows the products need a third of the time that the bytes need.
//
// P is rounded to the inputs' type for the second product (half a step relative to each term, as large as the rounding of the
// result); the sums stay in fp32 and add the unrounded values.

constexpr int kStreamRows = 16, kStreamKeys = 64, kStreamThreads = 160;

template <int D>
struct StreamCfg {
  static constexpr int kCtasPerSm = D == 256 ? 1 : 2;
  static constexpr int kTileBytes = kStreamKeys * D * 2;  // of K, and of V
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kBufLd = D + 8;  // padded: a quarter warp's 8-byte stores fall into distinct banks
  static constexpr int kSmemBytes = 1024 + kStages * 2 * kTileBytes + kStreamRows * kBufLd * 4 + 2 * 4 * kStreamRows * 4 + 256;
  static constexpr int kPieceFloats = kStreamRows * (D + 2);
};

// What block c of the join has to do: the segment that the start of CTA c's range cuts, if that is the first cut in it.
struct JoinRecord {
  int pieces;  // 0: nothing
  int b, hk, rg;
};

// The tiles of one sequence and its segments.
struct StreamSeq {
  Sequence s;
  int groups, tiles, sink_tiles, first_window_tile;
  int low;  // first position inside the first row's window
  __device__ int64_t weight(const Args& p) const { return int64_t(p.kv_heads) * groups * tiles; }
  __device__ int tile(int i) const { return i < sink_tiles ? i : first_window_tile + i - sink_tiles; }
};

__device__ __forceinline__ StreamSeq stream_seq(const Args& p, int b, int max_rows) {
  StreamSeq q;
  q.s = sequence_of(p, b);
  const int rows = q.s.rows * (p.heads / p.kv_heads);
  q.groups = rows <= max_rows ? (rows + kStreamRows - 1) / kStreamRows : 0;
  const int end = min(q.s.len, q.s.reach);
  q.low = p.window > 0 ? max(q.s.len - q.s.rows - p.window + 1, 0) : 0;
  q.sink_tiles = (min(min(p.sinks, q.low), end) + kStreamKeys - 1) / kStreamKeys;
  q.first_window_tile = max(q.low / kStreamKeys, q.sink_tiles);
  q.tiles = max(q.sink_tiles + max((end + kStreamKeys - 1) / kStreamKeys - q.first_window_tile, 0), 1);  // (1: zeros are written)
  return q;
}

// A walk over the segments from a position in the order of all tiles.
struct StreamCursor {
  int b, hk, rg, i;  // i: tile within the segment
  StreamSeq q;
  __device__ void next(const Args& p, int max_rows) {
    i = 0;
    if (++rg < q.groups) return;
    rg = 0;
    if (++hk < p.kv_heads) return;
    hk = 0;
    do b++; while (b < p.B && (q = stream_seq(p, b, max_rows)).groups == 0);
  }
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat162) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half2) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void stream_bar() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <typename T2, int D>
__global__ void __launch_bounds__(kStreamThreads, StreamCfg<D>::kCtasPerSm)
    attention_stream_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                            const __grid_constant__ Args p, int max_rows, float* pieces, JoinRecord* records, uint32_t* status) {
  using C = StreamCfg<D>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;  // the swizzle counts from 1024-byte boundaries
  uint8_t* smem = raw + (base - smem_u32(raw));
  float* buf = reinterpret_cast<float*>(smem + C::kStages * 2 * C::kTileBytes);
  float* warp_m = buf + kStreamRows * C::kBufLd;  // [4][16]
  float* warp_l = warp_m + 4 * kStreamRows;
  uint64_t* bars = reinterpret_cast<uint64_t*>(warp_l + 4 * kStreamRows);  // full[stages], empty[stages]
  __shared__ volatile uint32_t abort_flag;
  __shared__ int64_t sums[8];
  __shared__ int64_t start_base;
  __shared__ int start_b;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  auto full = [&](int s) { return smem_u32(bars + s); };
  auto empty = [&](int s) { return smem_u32(bars + C::kStages + s); };

  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::kStages; s++) mbar_init(full(s), 1), mbar_init(empty(s), 4);
    mbar_init_fence();
    prefetch_tensormap(&kmap), prefetch_tensormap(&vmap);
  }
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's range of the tiles -------------------------------------------------------------------------------
  int64_t mine = 0;
  for (int b = tid; b < p.B; b += kStreamThreads) mine += stream_seq(p, b, max_rows).weight(p);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) sums[warp] = mine;
  __syncthreads();
  const int64_t total = sums[0] + sums[1] + sums[2] + sums[3] + sums[4];
  const int64_t ctas = min(int64_t(gridDim.x), total), c = blockIdx.x;
  if (c >= ctas) {
    if (tid == 0) records[c].pieces = 0;
    return;
  }
  const int64_t t0 = total * c / ctas, t1 = total * (c + 1) / ctas;
  int64_t before = 0;  // tiles of the sequences before this round's
  if (tid == 0) start_b = -1;
  for (int b0 = 0; b0 < p.B; b0 += kStreamThreads) {
    const int b = b0 + tid;
    const int64_t w = b < p.B ? stream_seq(p, b, max_rows).weight(p) : 0;
    int64_t upto = w;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t round = 0;
    for (int i = 0; i < 5; i++) {
      if (i < warp) upto += sums[i];
      round += sums[i];
    }
    if (before + upto - w <= t0 && t0 < before + upto) start_b = b, start_base = before + upto - w;
    before += round;
    if (t0 < before) break;  // (t0 < total: some round holds it)
  }
  __syncthreads();
  if (start_b < 0) {  // (the lengths changed under the kernel: nothing is done)
    if (tid == 0) records[c].pieces = 0;
    return;
  }
  StreamCursor cur;
  cur.b = start_b, cur.q = stream_seq(p, cur.b, max_rows);
  {
    int64_t off = t0 - start_base;
    cur.i = int(off % cur.q.tiles), off /= cur.q.tiles;
    cur.rg = int(off % cur.q.groups), cur.hk = int(off / cur.q.groups);
  }
  if (tid == 0) {
    JoinRecord r = {0, cur.b, cur.hk, cur.rg};
    const int64_t s0 = t0 - cur.i, s1 = s0 + cur.q.tiles;
    if (cur.i > 0 && total * (c - 1) / ctas <= s0) r.pieces = int((s1 * ctas + total - 1) / total - 1 - c) + 2;
    records[c] = r;
  }

  if (warp == 4) {
    // ---- producer ----------------------------------------------------------------------------------------------------
    // Lane x looks up the page of box x of a tile, a tile ahead: the table's latency would add to the copy's.
    const int box = min(p.page_size, kStreamKeys), boxes = kStreamKeys / box;
    const uint32_t box_bytes = uint32_t(box) * 128u;  // per 64 channels
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool stop = false;  // a wait ran out (the same in all lanes)
    struct Box {
      int k0, page;
      bool need;
    };
    auto look_up = [&](const StreamCursor& at, int i) {
      const int reach = min(at.q.s.len, at.q.s.reach);
      Box x;
      x.k0 = at.q.tile(i) * kStreamKeys + lane * box, x.page = 0;
      x.need = lane < boxes && x.k0 < reach && (x.k0 < p.sinks || min(x.k0 + box, reach) > at.q.low);  // pages that no row sees are not read
      if (x.need) x.page = p.table[at.b * p.table_ld + x.k0 / p.page_size];
      return x;
    };
    Box next = look_up(cur, cur.i);
    for (int64_t t = t0; t < t1 && cur.b < p.B && !stop;) {
      const int end = int(min(int64_t(cur.q.tiles), cur.i + (t1 - t))), hk = cur.hk;
      if (cur.q.s.len > cur.q.s.reach && lane == 0) atomicCAS(status, 0u, uint32_t(kStatusBadPage));
      for (int i = cur.i; i < end; i++, t++) {
        const Box x = next;
        if (i + 1 < end) {
          next = look_up(cur, i + 1);
        } else {
          cur.next(p, max_rows);
          if (t + 1 < t1 && cur.b < p.B) next = look_up(cur, 0);
        }
        int page = x.page;
        if (x.need && (page < 0 || page >= p.pages)) page = p.pages, atomicCAS(status, 0u, uint32_t(kStatusBadPage));  // (reads zeros)
        const uint32_t needs = __ballot_sync(0xffffffffu, x.need);
        if (issued >= C::kStages && !warp_wait(empty(stage), phase ^ 1u, &abort_flag, status, kStatusEmptyWaitTimeout, 0)) {
          stop = true;
          break;
        }
        // one elected lane issues: copies issued by several lanes of a warp go out one lane at a time
        const uint32_t bar = full(stage), dst = base + stage * 2 * C::kTileBytes;
        const int key0 = __shfl_sync(0xffffffffu, x.k0, 0);
        if (elect_one()) mbar_arrive_expect_tx(bar, uint32_t(__popc(needs)) * 2 * (D / 64) * box_bytes);
        for (uint32_t left = needs; left; left &= left - 1) {
          const int lane_of = __ffs(left) - 1, page_of = __shfl_sync(0xffffffffu, page, lane_of), slot = (key0 + lane_of * box) & (p.page_size - 1);
          if (elect_one()) {
            const uint32_t kdst = dst + lane_of * box_bytes, vdst = kdst + C::kTileBytes;
#pragma unroll
            for (int d = 0; d < D / 64; d++) tma_load_4d(kdst + d * kStreamKeys * 128, &kmap, d * 64, slot, hk, page_of, bar);
#pragma unroll
            for (int d = 0; d < D / 64; d++) tma_load_4d(vdst + d * kStreamKeys * 128, &vmap, d * 64, slot, hk, page_of, bar);
          }
          __syncwarp();
        }
        issued++;
        if (++stage == C::kStages) stage = 0, phase ^= 1u;
      }
    }
    if (stop) {  // unwinding: no copy may still be in flight when the CTA ends
      for (int s = 0; s < C::kStages && s < issued; s++) {
        const int last = issued - 1 - ((issued - 1 - s) % C::kStages + C::kStages) % C::kStages;  // last use of ring place s
        uint32_t unused = 0;
        if (lane == 0) mbar_wait_bounded(full(s), uint32_t(last / C::kStages) & 1u, &abort_flag, &unused, kStatusDrainTimeout);
      }
    }
    return;
  }

  // ---- consumers -----------------------------------------------------------------------------------------------------
  const int G = p.heads / p.kv_heads, r0 = lane / 4, c2 = 2 * (lane % 4);
  const float to_log2 = p.scale * 1.4426950408889634f;
  const int my_key = warp * 16;
  // ldmatrix row addresses of this lane inside a 64-channel block: K (keys x 16 channels), V (transposed)
  const int krow = my_key + (lane / 16) * 8 + lane % 8, kchunk = (lane / 8) & 1;
  const int vrow = my_key + ((lane / 8) & 1) * 8 + lane % 8, vchunk = lane / 16;
  int stage = 0;
  uint32_t phase = 0;
  for (int64_t t = t0; t < t1 && cur.b < p.B; cur.next(p, max_rows)) {
    const StreamSeq& q = cur.q;
    const int from = cur.i, end = int(min(int64_t(q.tiles), from + (t1 - t)));
    const int total_rows = q.s.rows * G, reach = min(q.s.len, q.s.reach), first_pos = q.s.len - q.s.rows;
    // rows of this group: their positions, and their queries as the first product's left operand
    const int ra = cur.rg * kStreamRows + r0, rb = ra + 8;
    const int pos_a = ra < total_rows ? first_pos + ra / G : -1, pos_b = rb < total_rows ? first_pos + rb / G : -1;
    const int pmin = first_pos + cur.rg * kStreamRows / G, pmax = first_pos + (min((cur.rg + 1) * kStreamRows, total_rows) - 1) / G;
    uint32_t qf[D / 16][4];
    {
      const uint16_t* qa = static_cast<const uint16_t*>(p.q) + (q.s.row0 + ra / G) * p.q_ld_token + (cur.hk * G + ra % G) * p.q_ld_head + c2;
      const uint16_t* qb = static_cast<const uint16_t*>(p.q) + (q.s.row0 + rb / G) * p.q_ld_token + (cur.hk * G + rb % G) * p.q_ld_head + c2;
#pragma unroll
      for (int k = 0; k < D / 16; k++) {
        qf[k][0] = ra < total_rows ? *reinterpret_cast<const uint32_t*>(qa + 16 * k) : 0u;
        qf[k][1] = rb < total_rows ? *reinterpret_cast<const uint32_t*>(qb + 16 * k) : 0u;
        qf[k][2] = ra < total_rows ? *reinterpret_cast<const uint32_t*>(qa + 16 * k + 8) : 0u;
        qf[k][3] = rb < total_rows ? *reinterpret_cast<const uint32_t*>(qb + 16 * k + 8) : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;

    for (int i = from; i < end; i++, t++) {
      const bool here = warp_wait(full(stage), phase, &abort_flag, status, kStatusFullWaitTimeout, 0);
      const int k0 = q.tile(i) * kStreamKeys + my_key, k1 = k0 + 15;  // this warp's keys
      const bool some = k0 <= pmax && k0 < reach && (p.window == 0 || k1 > pmin - p.window || k0 < p.sinks);
      if (here && some) {
        const uint32_t kt = base + stage * 2 * C::kTileBytes, vt = kt + C::kTileBytes;
        float s[2][4] = {};
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
          uint32_t f[4];
          const int chunk = (k % 4) * 2 + kchunk;
          ldmatrix4(f, kt + (k / 4) * kStreamKeys * 128 + krow * 128 + ((chunk ^ (krow & 7)) << 4));
          mma16816(s[0], qf[k], f[0], f[1], T2{});
          mma16816(s[1], qf[k], f[2], f[3], T2{});
        }
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[n][e] *= to_log2;
        const bool all = k1 <= pmin && k1 < reach && (p.window == 0 || k0 > pmax - p.window || k1 < p.sinks);
        if (!all) {
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int j = k0 + n * 8 + c2 + (e & 1), pos = e < 2 ? pos_a : pos_b;
              const bool see = j <= pos && j < reach && (p.window == 0 || j > pos - p.window || j < p.sinks);
              if (!see) s[n][e] = -INFINITY;
            }
        }
        float x_a = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), x_b = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
        for (int d = 1; d < 4; d *= 2) {
          x_a = fmaxf(x_a, __shfl_xor_sync(0xffffffffu, x_a, d));
          x_b = fmaxf(x_b, __shfl_xor_sync(0xffffffffu, x_b, d));
        }
        if (__any_sync(0xffffffffu, x_a > m_a || x_b > m_b)) {  // a new maximum: what is there is scaled down to it
          const float n_a = fmaxf(m_a, x_a), n_b = fmaxf(m_b, x_b);
          const float f_a = n_a == -INFINITY ? 1.f : exp2f(m_a - n_a), f_b = n_b == -INFINITY ? 1.f : exp2f(m_b - n_b);
          m_a = n_a, m_b = n_b, l_a *= f_a, l_b *= f_b;
#pragma unroll
          for (int n = 0; n < D / 8; n++) o[n][0] *= f_a, o[n][1] *= f_a, o[n][2] *= f_b, o[n][3] *= f_b;
        }
        const float z_a = m_a == -INFINITY ? 0.f : m_a, z_b = m_b == -INFINITY ? 0.f : m_b;  // (a row that sees nothing yet)
#pragma unroll
        for (int n = 0; n < 2; n++) {
          s[n][0] = exp2f(s[n][0] - z_a), s[n][1] = exp2f(s[n][1] - z_a);
          s[n][2] = exp2f(s[n][2] - z_b), s[n][3] = exp2f(s[n][3] - z_b);
          l_a += s[n][0] + s[n][1], l_b += s[n][2] + s[n][3];
        }
        uint32_t pf[4];
        {
          T2 w[4];
          narrow(make_float2(s[0][0], s[0][1]), &w[0]), narrow(make_float2(s[0][2], s[0][3]), &w[1]);
          narrow(make_float2(s[1][0], s[1][1]), &w[2]), narrow(make_float2(s[1][2], s[1][3]), &w[3]);
#pragma unroll
          for (int e = 0; e < 4; e++) pf[e] = *reinterpret_cast<uint32_t*>(&w[e]);
        }
        // values of keys that no row of the group sees are whatever the cache holds there (0 x NaN would be NaN): cleared
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (!all) {
          auto any = [&](int j) { return j <= pmax && j < reach && (p.window == 0 || j > pmin - p.window || j < p.sinks); };
          keep0 = (any(k0 + c2) ? 0xffffu : 0u) | (any(k0 + c2 + 1) ? 0xffff0000u : 0u);
          keep1 = (any(k0 + c2 + 8) ? 0xffffu : 0u) | (any(k0 + c2 + 9) ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int n = 0; n < D / 8; n += 2) {
          uint32_t f[4];
          const int chunk = n % 8 + vchunk;
          ldmatrix4_trans(f, vt + (n / 8) * kStreamKeys * 128 + vrow * 128 + ((chunk ^ (vrow & 7)) << 4));
          if (!all) f[0] &= keep0, f[1] &= keep1, f[2] &= keep0, f[3] &= keep1;
          mma16816(o[n], pf, f[0], f[1], T2{});
          mma16816(o[n + 1], pf, f[2], f[3], T2{});
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(stage));
      if (++stage == C::kStages) stage = 0, phase ^= 1u;
    }

    // ---- the four warps' sums meet, in order ------------------------------------------------------------------------------
#pragma unroll
    for (int d = 1; d < 4; d *= 2) l_a += __shfl_xor_sync(0xffffffffu, l_a, d), l_b += __shfl_xor_sync(0xffffffffu, l_b, d);
    if (lane % 4 == 0) {
      warp_m[warp * kStreamRows + r0] = m_a, warp_m[warp * kStreamRows + r0 + 8] = m_b;
      warp_l[warp * kStreamRows + r0] = l_a, warp_l[warp * kStreamRows + r0 + 8] = l_b;
    }
    stream_bar();
    {
      float top_a = -INFINITY, top_b = -INFINITY;
      for (int w = 0; w < 4; w++) top_a = fmaxf(top_a, warp_m[w * kStreamRows + r0]), top_b = fmaxf(top_b, warp_m[w * kStreamRows + r0 + 8]);
      const float f_a = m_a == -INFINITY ? 0.f : exp2f(m_a - top_a), f_b = m_b == -INFINITY ? 0.f : exp2f(m_b - top_b);
      for (int w = 0; w < 4; w++) {
        if (w == warp) {
          float *ba = buf + r0 * C::kBufLd + c2, *bb = ba + 8 * C::kBufLd;
#pragma unroll
          for (int n = 0; n < D / 8; n++) {
            float2 va = make_float2(o[n][0] * f_a, o[n][1] * f_a), vb = make_float2(o[n][2] * f_b, o[n][3] * f_b);
            if (w > 0) {
              const float2 ua = *reinterpret_cast<float2*>(ba + 8 * n), ub = *reinterpret_cast<float2*>(bb + 8 * n);
              va.x += ua.x, va.y += ua.y, vb.x += ub.x, vb.y += ub.y;
            }
            *reinterpret_cast<float2*>(ba + 8 * n) = va, *reinterpret_cast<float2*>(bb + 8 * n) = vb;
          }
        }
        stream_bar();
      }
    }
    {
      const int r = tid / 8, part = tid % 8, row = cur.rg * kStreamRows + r;  // eight threads to a row
      float top = -INFINITY, l = 0.f;
      for (int w = 0; w < 4; w++) top = fmaxf(top, warp_m[w * kStreamRows + r]);
      for (int w = 0; w < 4; w++) l += warp_m[w * kStreamRows + r] == -INFINITY ? 0.f : warp_l[w * kStreamRows + r] * exp2f(warp_m[w * kStreamRows + r] - top);
      const float* src = buf + r * C::kBufLd;
      if (row < total_rows) {
        if (from == 0 && end == q.tiles) {
          store_row<T2, D, 8>(p, q.s.row0 + row / G, cur.hk * G + row % G, part, top, l, src);
        } else {  // cut: this CTA's piece of the segment (2 c: begun before this range; 2 c + 1: goes on after it)
          float* piece = pieces + (2 * c + (from > 0 ? 0 : 1)) * C::kPieceFloats;
          for (int d = part * 4; d < D; d += 32) *reinterpret_cast<float4*>(piece + r * D + d) = *reinterpret_cast<const float4*>(src + d);
          if (part == 0) piece[kStreamRows * D + r] = top, piece[kStreamRows * D + kStreamRows + r] = l;
        }
      }
    }
  }
}

// Joins the pieces of the cut segments: block (c, y) takes four rows of the segment whose first cut is the start of CTA c's
// range; four warps to a row, pieces dealt out to them in order.
template <typename T2, int D>
__global__ void __launch_bounds__(512) attention_join_kernel(const __grid_constant__ Args p, const float* pieces, const JoinRecord* records) {
  using C = StreamCfg<D>;
  __shared__ float part_m[4][4], part_l[4][4], acc[4][4][D];
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x;
  const JoinRecord r = records[c];
  if (r.pieces == 0) return;
  const Sequence s = sequence_of(p, r.b);
  const int G = p.heads / p.kv_heads, warp = threadIdx.x / 32, lane = threadIdx.x % 32, which = warp / 4, w = warp % 4;
  const int in_group = blockIdx.y * 4 + which, row = r.rg * kStreamRows + in_group;
  if (r.rg * kStreamRows + blockIdx.y * 4 >= s.rows * G) return;
  auto piece = [&](int i) { return pieces + int64_t(i == 0 ? 2 * (c - 1) + 1 : 2 * (c - 1 + i)) * C::kPieceFloats; };
  float m = -INFINITY, l = 0.f, o[D / 32] = {};
  if (row < s.rows * G) {
    for (int i = w; i < r.pieces; i += 4) m = fmaxf(m, piece(i)[kStreamRows * D + in_group]);
#pragma unroll 4
    for (int i = w; i < r.pieces; i += 4) {
      const float* x = piece(i);
      const float mi = x[kStreamRows * D + in_group], f = mi == -INFINITY ? 0.f : exp2f(mi - m);
      l += f * x[kStreamRows * D + kStreamRows + in_group];
#pragma unroll
      for (int e = 0; e < D / 32; e++) o[e] += f * x[in_group * D + e * 32 + lane];
    }
  }
  if (lane == 0) part_m[which][w] = m, part_l[which][w] = l;
  __syncthreads();
  float top = -INFINITY;
  for (int i = 0; i < 4; i++) top = fmaxf(top, part_m[which][i]);
  const float f = m == -INFINITY ? 0.f : exp2f(m - top);
#pragma unroll
  for (int e = 0; e < D / 32; e++) acc[which][w][e * 32 + lane] = o[e] * f;
  __syncthreads();
  if (w > 0 || row >= s.rows * G) return;
  l = 0.f;
  for (int i = 0; i < 4; i++) l += part_m[which][i] == -INFINITY ? 0.f : part_l[which][i] * exp2f(part_m[which][i] - top);
#pragma unroll
  for (int e = 0; e < D / 32; e++) {
    const int d = e * 32 + lane;
    acc[which][0][d] = acc[which][0][d] + acc[which][1][d] + acc[which][2][d] + acc[which][3][d];
  }
  __syncwarp();
  store_row<T2, D, 32>(p, s.row0 + row / G, r.hk * G + row % G, lane, top, l, acc[which][0]);
}

// Scratch of a launch: the records, then the pieces.
template <int D>
size_t stream_scratch_bytes(int ctas) {
  return (size_t(ctas) * sizeof(JoinRecord) + 255) / 256 * 256 + size_t(ctas) * 2 * StreamCfg<D>::kPieceFloats * 4;
}

template <typename T2, int D>
int launch_stream(const Args& p, int max_rows, void* ws, cudaStream_t s, uint32_t* status) {
  using C = StreamCfg<D>;
  auto kernel = attention_stream_kernel<T2, D>;
  static bool done[64] = {};
  int dev = 0;
  Q27B_CUDA(cudaGetDevice(&dev));
  if (!(dev < 64 && done[dev])) {
    Q27B_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    if (dev < 64) done[dev] = true;
  }
  CUtensorMap km, vm;
  const int box = std::min(p.page_size, kStreamKeys);
  if (int rc = make_cache_map(&km, p, p.k_cache, p.kc_ld_page, p.kc_ld_head, p.kc_ld_slot, box)) return rc;
  if (int rc = make_cache_map(&vm, p, p.v_cache, p.vc_ld_page, p.vc_ld_head, p.vc_ld_slot, box)) return rc;
  const int ctas = C::kCtasPerSm * sm_count();
  JoinRecord* records = static_cast<JoinRecord*>(ws);
  float* pieces = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + (size_t(ctas) * sizeof(JoinRecord) + 255) / 256 * 256);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas)), cfg.blockDim = dim3(kStreamThreads), cfg.dynamicSmemBytes = C::kSmemBytes, cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 1 : 0;
  Q27B_CUDA(cudaLaunchKernelEx(&cfg, kernel, km, vm, p, max_rows, pieces, records, status));
  cfg.gridDim = dim3(unsigned(ctas), kStreamRows / 4), cfg.blockDim = dim3(512), cfg.dynamicSmemBytes = 0;
  Q27B_CUDA(cudaLaunchKernelEx(&cfg, attention_join_kernel<T2, D>, p, static_cast<const float*>(pieces), static_cast<const JoinRecord*>(records)));
  return 0;
}
