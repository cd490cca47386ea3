// Paged decode attention over a 4-bit KV cache. Part of decode_attention.cu (included there, inside
// its namespace): the plan, the workspace, the split merge and the order of launches are those of
// the 16-bit kernel; what differs is how a worker warp fetches and computes a tile.
//
//   * A (block, head) tile of keys, values and pairs (int4_tile.cuh) is 2304 contiguous bytes: one
//     untiled bulk copy a tile, up to kStages of them ahead of the compute in each warp's ring.
//   * No element is dequantised. With K = s c + m per (token, group) and c a whole number 0..15,
//       q . K = sum over groups of  s (q . c) + m (sum of q)
//       sum_t p_t V_t = sum_t (p_t s_t) c_t + sum_t p_t m_t
//     so the codes go to the tensor cores as they are, exactly, and scales and minima meet them
//     in fp32.
//   * A code becomes a bf16 number with one AND: a nibble under a zero exponent is the subnormal c * 2^-133,
//     or c * 2^-129 four bits further up (bf16's least normal binade has the spacing of its subnormals),
//     exact on the tensor cores; the other operand carries a power of two that keeps the products within
//     fp32's range. Beside fp16 queries, whose 11 bits bf16 does not hold, a key code is an fp16 number: a
//     nibble under the exponent of 64 reads as 64 + c, and the constant is taken out with the keys' minima
//     (m - 64 s in place of m) in fp32.
//   * S^T = K Q^T as in the 16-bit kernel (16 tokens x 8 heads of the group, m16n8k16), in the queries' type.
//     A lane's codes of a token are one 16-byte load; which dim sits where in the contraction is free as
//     long as the query fragments follow.
//   * O^T += V^T P^T in bf16: P * s, made in fp32, goes in as two bf16 parts (16 bits), each with the whole
//     range of fp32's exponents, so that neither a token's nor a group's scale costs another one bits.
//     Token pairs share a 32-bit word, so that the transposed fragment comes out of the AND without a
//     transposing load. sum p m is 4 FMAs a token and lane.
//   * The tensor cores cut off what an addition pushes out of the accumulator, always downwards, so a sum
//     of one sign drifts with its length. So odd tokens count from the top: with -P s they meet 15 - c (the
//     AND's result with those four bits turned over, the same instruction), sum p (m + 15 s) in place of
//     their sum p m makes up for it, and O stays near 0.
//   * The running maximum moves only when a score exceeds it by kSlack (log2 units): sums are fp32, and
//     most tiles need one vote instead of a reduction over the tokens and a rescaling of O.
//   * One warp of the CTA requests the tiles of all others, a lane for each, so that walking the units
//     and the block table costs the computing warps neither instructions nor registers.
//
// What it takes, per layer inside a graph of layers (the 16-bit kernel on the same lengths), and with the layer's
// cache write before each attention, as a decode step has it (the 16-bit kernels likewise):
//   4 sequences of 17..300 tokens, 28/4 heads fp16       7.6 us (6.9)    9.5 us (7.9)
//   64 of lognormal(5.5, 1) tokens, 28/4 heads fp16     10.5 us (12.3)  13.7 us (13.7)
//   256 of lognormal(6, 1) tokens, 32/4 heads bf16      33.7 us (55.6)  38.4 us (57.0)  2.5 TB/s of K/V
//   2 of 40,001..65,535 tokens, 32/4 heads bf16         27.7 us (48.3)  29.2 us (49.8)
//   16 of 2048..4096 tokens, 40/40 heads fp16           79.0 us (178)   84.3 us (182)   3.7 TB/s
// What bounds it: walking the units, requesting nothing and computing nothing, start and merge included, took
// 20.5 us of the fourth, 23.4 of the third and 37.2 of the last; requesting the tiles without computing 25.7,
// 29.3 and 60.5. So the requesting warp's loop, one 2304-byte tile a step for each worker, uses up most of the
// time the memory would need (85 clocks a tile and SM, of 100 for its bytes). Beside it the work per byte is
// 3.6 times that of the 16-bit kernel, ~350 instructions a tile at half the issue rate (three warps a
// scheduler, 168 registers each). 15 workers of 128 registers, 7 of 255, two tiles at a time in a worker,
// the next tile's scores ahead of this one's products, 16 % fewer integer instructions: each within 5 % or
// slower. Workers that issue their own copies, from a queue of addresses that the spare warp fills, took
// 94 us for the last case, 38 for the third. P * scale in one fp16 number, of 11 bits under one power of two
// for both groups, took 1 to 3 % less, and gave wrong values where scales lie far apart.

template <int NT>
struct Int4Smem {
  // Worker warps (the plan's workers) and one warp that requests their tiles, one lane a worker.
  static constexpr int kWarps = NT == 1 ? 11 : 7;
  static constexpr int kThreads = (kWarps + 1) * 32;
  static constexpr int kStages = NT == 1 ? 8 : 11;
  static constexpr int kMergeLoads = NT == 1 ? 8 : kMergeBatch;  // pieces of a merge in flight per lane
  static constexpr int kQSlot = 8 * NT * kHeadDim * 2;
  static constexpr int kRing = kStages * kInt4TileBytes;
  static constexpr int kPerWarp = kRing + kQSlot;
  // Per worker: barriers (tile landed / free for each stage, queries landed / free), tokens of each
  // stage's tile, and the record of the unit whose queries lie in the slot.
  static constexpr int kBars = 2 * kStages + 2;
  static constexpr int kTokens = 8 * kBars;
  static constexpr int kRecord = (kTokens + 4 * kStages + 15) / 16 * 16;
  static constexpr int kMeta = kRecord + 32;
  static constexpr int kOffMeta = kWarps * kPerWarp;
  static constexpr int kOffDone = kOffMeta + kWarps * kMeta;     // workers that have published
  static constexpr size_t kDynamic = size_t(kOffDone) + 16 + 128;  // + alignment slack
  static_assert(kPerWarp % 128 == 0 && kDynamic <= 232448, "ring alignment and capacity");
};

// (x & mask) | bits in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
  return r;
}
// Nibbles k and k + 4 (k = 0..3) of a key word as fp16 pairs, code + kBias, into a[k]. Under the exponent of
// 64 a nibble at mantissa bits 4..7 reads as 64 + c and one at bits 0..3 as 64 + c / 16, which one
// packed FMA (16 x - 960, exact) turns into 64 + c: that leaves one shift for two nibbles, as the
// integer pipe, half as wide as the FMA pipe, is the busier one.
constexpr float kBias = 64.f;
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t (&a)[4]) {
  const __half2 k16 = __float2half2_rn(16.f), k960 = __float2half2_rn(-960.f);
  auto up = [&](uint32_t x) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), k16, k960);
    return *reinterpret_cast<const uint32_t*>(&r);
  };
  const uint32_t t = w >> 8;
  a[0] = up(and_or(w, 0x000f000fu, 0x54005400u));
  a[1] = and_or(w, 0x00f000f0u, 0x54005400u);
  a[2] = up(and_or(t, 0x000f000fu, 0x54005400u));
  a[3] = and_or(t, 0x00f000f0u, 0x54005400u);
}
// The same nibbles as bf16 pairs: a[0], a[2] hold code * 2^-133, a[1], a[3] code * 2^-129; of values the upper
// halves, which are odd tokens, 15 - code.
template <bool kTurn>
__device__ __forceinline__ void code_pairs_bf16(uint32_t w, uint32_t (&a)[4]) {
  const uint32_t t = w >> 8, low = kTurn ? 0x000f0000u : 0u, high = kTurn ? 0x00f00000u : 0u;
  a[0] = (w & 0x000f000fu) ^ low;
  a[1] = (w & 0x00f000f0u) ^ high;
  a[2] = (t & 0x000f000fu) ^ low;
  a[3] = (t & 0x00f000f0u) ^ high;
}
// What bf16 queries, brought to 1 by a power of two, are held times (1 / 16 of it where they meet a[1], a[3]); the
// products with the codes are then times 2^-13.
constexpr float kQueryTop = 0x1p120f;
// 2^n, -126 <= n <= 127.
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float(static_cast<uint32_t>(n + 127) << 23); }
// Two fp32 numbers as pairs of bf16: the upper 8 bits of each cut off, and the rest rounded to 8.
__device__ __forceinline__ void split2(float y0, float y1, uint32_t& hi, uint32_t& lo) {
  const uint32_t b0 = __float_as_uint(y0), b1 = __float_as_uint(y1);
  hi = __byte_perm(b0, b1, 0x7632);
  lo = pack2<__nv_bfloat16>(y0 - __uint_as_float(b0 & 0xffff0000u), y1 - __uint_as_float(b1 & 0xffff0000u));
}
// What P * scale is held times. fp16's scales, 2^-24 to 2^13, go with this one number; over bf16's range it
// follows the largest finite scale met, which it brings to 2^96 or up to 2^17 times that (2^127 is its own end).
// Products and sums then stay below 2^11, and the 16 bits of a scale 2^-96 of the largest above fp32's last.
constexpr float kTop = 0x1p96f;
constexpr uint32_t kScaleInf = 0x7f80u;   // bits of a bf16 infinity
constexpr float kScaleLeast = 0x1p-31f;   // smaller scales count as this
constexpr uint32_t kScaleRoom = 0x087fu;  // added to a scale's exponent: the largest one with the same factor

// Products, transpositions and shared loads that the compiler may move among one another (those of
// aeg_common.cuh are volatile and keep their order): a tile's chains overlap only if it does. The
// loads stay behind the barrier waits, which clobber memory.
template <typename T>
__device__ __forceinline__ void mma_free(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_free(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// Whether the phase with the given parity has completed; does not wait.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ int atom_add_acq_rel_cta(int* p, int v) {
  int old;
  asm volatile("atom.acq_rel.cta.shared::cta.add.s32 %0, [%1], %2;" : "=r"(old) : "r"(smem_u32(p)), "r"(v) : "memory");
  return old;
}
__device__ __forceinline__ uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint2 lds64(const uint8_t* p) { return *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ void bulk_load_1d_hint(void* smem_dst, const void* gmem_src, uint32_t bytes, uint64_t* bar,
                                                  uint64_t l2_policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(gmem_src)), "r"(bytes), "r"(smem_u32(bar)), "l"(l2_policy)
      : "memory");
}

// A worker's part of shared memory.
template <int NT>
struct Int4Worker {
  using SL = Int4Smem<NT>;
  uint8_t* ring;
  uint8_t* q;
  uint64_t* full;   // tile landed
  uint64_t* empty;  // stage free
  uint64_t* qfull;
  uint64_t* qempty;
  int* tokens;      // valid tokens of the stage's tile
  int4* record;     // {tiles (-1: no more units), partial slot or -1, sequence, KV head}
  volatile uint32_t* seen;
  __device__ Int4Worker(uint8_t* smem, int w) {
    ring = smem + w * SL::kPerWarp;
    q = ring + SL::kRing;
    uint8_t* meta = smem + SL::kOffMeta + w * SL::kMeta;
    full = reinterpret_cast<uint64_t*>(meta);
    empty = full + SL::kStages;
    qfull = empty + SL::kStages;
    qempty = qfull + 1;
    tokens = reinterpret_cast<int*>(meta + SL::kTokens);
    record = reinterpret_cast<int4*>(meta + SL::kRecord);
    seen = reinterpret_cast<uint32_t*>(meta + SL::kRecord + 16);
  }
};

// A worker's range of units and its first unit's record; an empty range if the plan does not fit this
// launch. `report` says whether the caller reports that.
struct Int4Range {
  int u_beg, u_end;
  int4 ra, rb;
};
__device__ __forceinline__ Int4Range int4_range(const AttnParams& p, int gw, int total_warps, bool report) {
  const uint64_t keep = l2_policy_evict_last();
  Int4Range r;
  r.u_beg = ld_hint(&p.ws.warp_rec[3 * gw].x, keep);
  r.ra = ld_hint(&p.ws.warp_rec[3 * gw + 1], keep);
  r.rb = ld_hint(&p.ws.warp_rec[3 * gw + 2], keep);
  r.u_end = ld_hint(&p.ws.warp_rec[3 * (gw + 1)].x, keep);
  const int planned_warps = ld_hint(&p.ws.header[kHdrWarps], keep);
  const int planned_units = ld_hint(&p.ws.header[kHdrUnits], keep);
  if (!(planned_warps == total_warps && planned_units <= p.max_units && r.u_beg >= 0 && r.u_beg <= r.u_end &&
        r.u_end <= planned_units)) {
    if (report && r.u_beg != r.u_end) atomicOr(&g_deverr_attn, AEG_DEVERR_PLAN_MISMATCH);
    r.u_end = r.u_beg;
  }
  return r;
}

// The requesting warp: lane w walks worker w's units (their records and queries) and tiles. Block ids
// come four at a time and four tiles ahead, unit records one unit ahead, so that no step waits for a
// load it has just made (with ids two tiles ahead every step did, and streaming took 1.1 to 1.2 times
// as long). A worker's first unit's record and queries are not among them: the worker fetches those
// itself, beside the first tiles. Without a tensor map there is no zero fill: a tile whose id is
// outside the pool is not fetched and has no valid tokens.
template <typename T, int NT>
__device__ __forceinline__ void request_tiles(const AttnParams& p, uint8_t* smem, int lane) {
  using SL = Int4Smem<NT>;
  const uint64_t keep = l2_policy_evict_last(), pol = l2_policy_evict_first();
  const bool worker = lane < SL::kWarps;
  const Int4Worker<NT> w(smem, worker ? lane : 0);
  const int gw = static_cast<int>(blockIdx.x) * SL::kWarps + (worker ? lane : 0);

  // The plan and the first tiles come before the wait for the preceding kernel only where the host
  // knows that it wrote neither.
  const bool early = p.plan_ready && p.prefetch_kv;
  const int total_warps = static_cast<int>(gridDim.x) * SL::kWarps;
  Int4Range range;
  if (p.plan_ready) range = int4_range(p, gw, total_warps, worker);
  if (!early) pdl_wait_primary();
  if (!p.plan_ready) range = int4_range(p, gw, total_warps, worker);
  const int u_end = range.u_end;
  int4 ra = range.ra, rb = range.rb;

  // Tiles: unit ut (its record in ra, rb), tile i of n, the ids of the tiles from i on that are at hand
  // (the first `at_hand` of c) and those after them (d); the next unit's record.
  int ut = range.u_beg, i = 0, n = 0, n_ctx = 0, at_hand = 0;
  int4 c = make_int4(0, 0, 0, 0), d = c;
  const int* ids = p.tables;  // of the first tile in d
  const T* tiles = static_cast<const T*>(p.k_cache);
  int4 na = make_int4(0, 0, 0, -1), nb = make_int4(0, 0, 0, 0);
  auto load_ids = [&](int left) {  // of up to `left` tiles
    if (left > 0) d.x = ids[0];
    if (left > 1) d.y = ids[1];
    if (left > 2) d.z = ids[2];
    if (left > 3) d.w = ids[3];
  };
  auto enter = [&]() {  // begins unit ut
    n = ut < u_end ? unit_items(ra, rb, p) : 0;
    i = 0;
    if (ut < u_end) {
      c = make_int4(rb.y, rb.z, rb.w, 0);
      at_hand = 3;
      n_ctx = rb.x - ra.y * kBlockTokens;
      ids = p.tables + static_cast<int64_t>(ra.x / p.Hkv) * p.table_stride + ra.y + 3;
      load_ids(n - 3);
      tiles = static_cast<const T*>(p.k_cache) + static_cast<int64_t>(ra.x % p.Hkv) * kInt4TileElems;
      if (ut + 1 < u_end) {
        na = ld_hint(&p.ws.units[2 * (ut + 1)], keep);
        nb = ld_hint(&p.ws.units[2 * (ut + 1) + 1], keep);
      }
    }
  };
  enter();
  // Queries: unit uq, its record (that of the second unit, the first one's being the worker's own).
  int uq = ut + 1;
  int4 qa = na, qb = nb;

  uint32_t st = 0, ph = 1, qph = 1;  // a barrier that has completed no phase counts as free
  auto tile_step = [&]() -> bool {
    if (i >= n) {
      if (ut >= u_end) return false;
      ++ut;
      ra = na;
      rb = nb;
      enter();
      return true;
    }
    if (!mbar_test(&w.empty[st], ph)) return false;
    if (at_hand == 0) {
      c = d;
      at_hand = 4;
      ids += 4;
      load_ids(n - i - 4);
    }
    const int id = c.x;
    c = make_int4(c.y, c.z, c.w, 0);
    --at_hand;
    const bool inside = static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks);
    w.tokens[st] = inside ? min(kBlockTokens, n_ctx - i * kBlockTokens) : 0;
    if (inside) {
      mbar_arrive_expect_tx(&w.full[st], kInt4TileBytes);
      bulk_load_1d_hint(w.ring + st * kInt4TileBytes, tiles + static_cast<int64_t>(id) * p.block_stride, kInt4TileBytes,
                        &w.full[st], pol);
    } else {
      atomicOr(&g_deverr_attn, AEG_DEVERR_BLOCK_ID_RANGE);
      mbar_arrive(&w.full[st]);
    }
    ++i;
    if (++st == SL::kStages) {
      st = 0;
      ph ^= 1;
    }
    return true;
  };
  if (early) {
    if (worker)
      for (int k = 0; k < SL::kStages + 2; ++k) tile_step();
    __syncwarp();
    pdl_wait_primary();
  }

  bool run = worker, more_units = worker;
  uint64_t idle_since = 0;
  while (__any_sync(0xffffffffu, run)) {
    bool moved = false;
    if (run) {
      if (more_units && mbar_test(w.qempty, qph)) {
        const int tiles_q = uq < u_end ? unit_items(qa, qb, p) : -1;
        const int b = qa.x / p.Hkv, h = qa.x % p.Hkv;
        if (tiles_q == 0) {  // a record that does not fit this call: left out, by the walk over tiles too
          atomicOr(&g_deverr_attn, AEG_DEVERR_PLAN_MISMATCH);
        } else {
          *w.record = make_int4(tiles_q, qa.w, b, h);
          if (tiles_q > 0 && p.q_bulk) {
            const uint32_t bytes = p.G * kHeadDim * 2;
            mbar_arrive_expect_tx(w.qfull, bytes);
            bulk_load_1d(w.q, static_cast<const T*>(p.q) + static_cast<int64_t>(b) * p.q_stride +
                                  static_cast<int64_t>(h) * p.G * kHeadDim, bytes, w.qfull);
          } else {
            mbar_arrive(w.qfull);
          }
          qph ^= 1;
        }
        more_units = tiles_q >= 0;
        ++uq;
        if (uq < u_end) {
          qa = ld_hint(&p.ws.units[2 * uq], keep);
          qb = ld_hint(&p.ws.units[2 * uq + 1], keep);
        }
        moved = true;
      }
      if (tile_step()) {
        moved = true;
        tile_step();
      }
      run = more_units || ut < u_end;
    }
    if (__any_sync(0xffffffffu, moved)) {
      idle_since = 0;
    } else {
      const uint64_t now = globaltimer_ns();
      if (idle_since == 0) idle_since = now;
      if (now - idle_since > kWaitLimitNs) {
        if (lane == 0) atomicOr(&g_deverr_attn, AEG_DEVERR_WAIT_TIMEOUT);
        return;
      }
      __nanosleep(40);
    }
  }
}

template <typename T, int NT>
__global__ void __launch_bounds__(Int4Smem<NT>::kThreads, 1) decode_attn_int4_kernel(const AttnParams p) {
  using SL = Int4Smem<NT>;
  constexpr int kW = SL::kWarps, kSt = SL::kStages;
  constexpr float kNoMax = -3e38f;  // the running maximum before the first score, below all but infinite ones
  constexpr float kSlack = 6.f;     // scores may exceed the running maximum by this (log2 units)

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 127) & ~127u) - raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  int* const done = reinterpret_cast<int*>(smem + SL::kOffDone);
  if (threadIdx.x == 0) *done = 0;
  if (warp < kW && lane == 0) {
    const Int4Worker<NT> w(smem, warp);
    for (int s = 0; s < SL::kBars; ++s) mbar_init(&w.full[s], 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (warp == kW) {
    request_tiles<T, NT>(p, smem, lane);
    return;
  }

  const Int4Worker<NT> wk(smem, warp);
  const uint8_t* const ring = wk.ring;
  const int gw = static_cast<int>(blockIdx.x) * kW + warp;
  const int G = p.G;
  const int total_warps = static_cast<int>(gridDim.x) * kW;
  const uint64_t keep = l2_policy_evict_last();
  T* out = static_cast<T*>(p.out);
  const int quad = lane & 3;  // column pair of the accumulator fragment
  const int grp = lane >> 2;  // row of the accumulator fragment
  Int4Range range;
  if (p.plan_ready) range = int4_range(p, gw, total_warps, false);
  pdl_wait_primary();
  pdl_launch_dependents();
  if (!p.plan_ready) range = int4_range(p, gw, total_warps, false);

  // This warp's share of the split merge and the launches with this plan so far (see
  // decode_attn_kernel); needed when its units are done.
  int4 mr = make_int4(0, 0, 0, 0);
  if (lane == 0) mr = ld_hint(&p.ws.merge_rec[gw], keep);
  else if (lane == 1) mr.x = ld_hint(&p.ws.header[kHdrWarps], keep);
  else if (lane == 2) mr.x = ld_hint(&p.ws.header[kHdrSplitPairs], keep);
  else if (lane == 3) mr.x = ld_relaxed_gpu(&p.ws.warp_flag[gw * kFlagStride]);

  bool lost = false;  // a wait ran out (the lanes agree on it): this warp's results are not complete
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, kWaitLimitNs))) {
      if (lane == 0) atomicOr(&g_deverr_attn, AEG_DEVERR_WAIT_TIMEOUT);
      lost = true;
    }
  };
  uint32_t st_con = 0, ph_con = 0, q_phase = 0;

  // The first unit's record comes from the plan and its queries from global memory; later ones through
  // shared memory, from the requesting warp.
  bool first = range.u_beg < range.u_end;
  while (!lost) {
    int n, slot, b, h;
    if (first) {
      n = unit_items(range.ra, range.rb, p);
      slot = range.ra.w;
      b = range.ra.x / p.Hkv;
      h = range.ra.x % p.Hkv;
      if (n == 0) {
        if (lane == 0) atomicOr(&g_deverr_attn, AEG_DEVERR_PLAN_MISMATCH);
        first = false;
        continue;
      }
    } else {
      wait(wk.qfull, q_phase);
      if (lost) break;
      q_phase ^= 1;
      const int4 rec = *wk.record;
      n = rec.x;
      slot = rec.y;
      b = rec.z;
      h = rec.w;
      if (n < 0) break;
    }

    // A negative scale goes into the sign of q, so that larger sums always mean larger scores. bf16
    // queries are brought to 1 by a power of two of the head's own, 2^-a, which returns with the scale of the
    // scores: exactly, down to elements 2^-110 of the head's largest. Half of it, of the group's largest head,
    // goes to the keys (2^(a / 2 - 8)): then large queries with small keys and small queries with large keys
    // both leave the unscaled scores in fp32's range.
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    uint32_t qf[NT][8][2];
    float qs[NT][2][2];  // [column][group]
    float sc[NT][2];     // scores to log2 units [column]
    int e_top = 1;       // exponent of the group's largest finite |q|
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + grp;
      uint32_t xw[4][4];
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        const T* src = static_cast<const T*>(p.q) + static_cast<int64_t>(b) * p.q_stride +
                       (static_cast<int64_t>(h) * G + head) * kHeadDim + w * 32 + quad * 8;
        if (head < G) {
          if (!p.q_bulk) {  // rows that are not 16-byte aligned
            const uint32_t* s4 = reinterpret_cast<const uint32_t*>(src);
            x = make_uint4(s4[0], s4[1], s4[2], s4[3]);
          } else if (first) {
            x = *reinterpret_cast<const uint4*>(src);
          } else {
            x = lds128(wk.q + head * (kHeadDim * 2) + w * 64 + quad * 16);
          }
        }
        xw[w][0] = x.x ^ flip;
        xw[w][1] = x.y ^ flip;
        xw[w][2] = x.z ^ flip;
        xw[w][3] = x.w ^ flip;
        if constexpr (!std::is_same<T, __half>::value)
          for (int i = 0; i < 4; ++i) top = __vmaxu2(top, xw[w][i] & 0x7fff7fffu);
      }
      float back = 1.f, sum[2] = {0.f, 0.f};
      if constexpr (!std::is_same<T, __half>::value) {
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = static_cast<int>(max(top & 0xffffu, top >> 16) >> 7);  // exponent of the largest |q|
        if (e < 255) e_top = max(e_top, e);
        const int ef = min(max(254 - e, 1), 253);
        const float to = __uint_as_float(static_cast<uint32_t>(ef) << 23);  // 2^(127 - e): |q| below 2
        back = __uint_as_float(static_cast<uint32_t>(254 - ef) << 23);
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(xw[w][i]);
            const float x = f.x * to, y = f.y * to;
            sum[w >> 1] += x + y;
            xw[w][i] = pack2<T>(x * kQueryTop, y * (kQueryTop / 16.f));
          }
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(xw[w][i]);
            sum[w >> 1] += f.x + f.y;
          }
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        qf[nt][2 * w][0] = __byte_perm(xw[w][0], xw[w][2], 0x5410);
        qf[nt][2 * w][1] = __byte_perm(xw[w][0], xw[w][2], 0x7632);
        qf[nt][2 * w + 1][0] = __byte_perm(xw[w][1], xw[w][3], 0x5410);
        qf[nt][2 * w + 1][1] = __byte_perm(xw[w][1], xw[w][3], 0x7632);
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        qs[nt][0][g] = __shfl_sync(0xffffffffu, sum[g], 8 * quad);
        qs[nt][1][g] = __shfl_sync(0xffffffffu, sum[g], 8 * quad + 4);
      }
      sc[nt][0] = __shfl_sync(0xffffffffu, back, 8 * quad);
      sc[nt][1] = __shfl_sync(0xffffffffu, back, 8 * quad + 4);
    }
    float key_unit = 1.f;  // times the keys' scales
    if constexpr (!std::is_same<T, __half>::value) {
      e_top = __reduce_max_sync(0xffffffffu, e_top);
      const int w = ((e_top - 127) >> 1) - 8;
      key_unit = power_of_two(w + 13);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sc[nt][i] *= power_of_two(-w);
          qs[nt][i][0] *= power_of_two(w);
          qs[nt][i][1] *= power_of_two(w);
        }
    }
    // Not 0, so that -infinity stays below all scores, nor infinite, so that the largest keeps its weight.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[nt][i] = fminf(fmaxf(sc[nt][i] * fabsf(p.scale_log2), 1e-37f), 3e38f);
    // The slot is free once every lane's values have arrived: the vote stored before the arrival needs
    // them all.
    if (!first) {
      uint32_t dep = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) dep |= qf[nt][ks][0] | qf[nt][ks][1];
      const uint32_t any = __ballot_sync(0xffffffffu, dep != 0);
      if (lane == 0) {
        *wk.seen = any;
        mbar_arrive(wk.qempty);
      }
    }
    first = false;

    // Running maximum of the unscaled scores and the score from which it moves (rounded down: p stays
    // within 2^kSlack however coarse the scores are); sum of p; sum of p * (what code 0 stands for)
    // [column][group]. O is held times |vmul|, which has the sign of this lane's tokens.
    float o[8][NT][4];
    float m[NT][2], mt_[NT][2], l[NT][2], om[NT][2][2];
    const bool odd = grp & 1;
    const float code0 = odd ? 15.f : 0.f;
    float vmul = odd ? -kTop : kTop;
    uint32_t vlim = 0;  // bits of the largest scale allowed for (bf16)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[nt][i] = kNoMax;
        mt_[nt][i] = __fadd_rd(kNoMax, kSlack / sc[nt][i]);
        l[nt][i] = om[nt][i][0] = om[nt][i][1] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.f;
    }
    // Scores of the tile in stage `st`, unscaled: S^T, one accumulator per group; rows are tokens grp
    // and grp + 8.
    auto scores = [&](uint32_t st, float (*x)[4]) {
      const uint8_t* tile = ring + st * kInt4TileBytes;
      const uint4 kc0 = lds128(tile + grp * 64 + quad * 16), kc1 = lds128(tile + 512 + grp * 64 + quad * 16);
      const uint2 kp0 = lds64(tile + kInt4KeyPairs + grp * 8), kp1 = lds64(tile + kInt4KeyPairs + 64 + grp * 8);
      const uint32_t kw0[4] = {kc0.x, kc0.y, kc0.z, kc0.w}, kw1[4] = {kc1.x, kc1.y, kc1.z, kc1.w};
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int w = 2 * g; w < 2 * g + 2; ++w) {
          uint32_t lo[4], hi[4];
          if constexpr (std::is_same<T, __half>::value) {
            code_pairs(kw0[w], lo);
            code_pairs(kw1[w], hi);
          } else {
            code_pairs_bf16<false>(kw0[w], lo);
            code_pairs_bf16<false>(kw1[w], hi);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t a[4] = {lo[2 * u], hi[2 * u], lo[2 * u + 1], hi[2 * u + 1]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_free<T>(s[nt], a, qf[nt][2 * w + u][0], qf[nt][2 * w + u][1]);
          }
        }
        float2 f0 = unpack2<T>(g == 0 ? kp0.x : kp0.y), f1 = unpack2<T>(g == 0 ? kp1.x : kp1.y);
        float b0 = f0.y, b1 = f1.y;
        if constexpr (std::is_same<T, __half>::value) {
          b0 = fmaf(-kBias, f0.x, b0);
          b1 = fmaf(-kBias, f1.x, b1);
        } else {
          f0.x *= key_unit;
          f1.x *= key_unit;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x[nt][i] = fmaf(f0.x, s[nt][i], g == 0 ? b0 * qs[nt][i][g] : fmaf(b0, qs[nt][i][g], x[nt][i]));
            x[nt][i + 2] = fmaf(f1.x, s[nt][i + 2], g == 0 ? b1 * qs[nt][i][g] : fmaf(b1, qs[nt][i][g], x[nt][i + 2]));
          }
      }
    };

    // Makes room for the scores x and the scales of the value pairs vp0, vp1: the maxima move to the tile's,
    // and what was summed so far follows.
    auto make_room = [&](const float (*x)[4], const uint2& vp0, const uint2& vp1) {
      float grow = 1.f;
      if constexpr (!std::is_same<T, __half>::value) {
        // Of the finite scales alone: NaN needs no room, it makes its own group's result NaN by itself, and
        // the other group of the head goes on.
        uint32_t top = 0;
        for (const uint32_t pair : {vp0.x, vp0.y, vp1.x, vp1.y}) {
          const uint32_t scale = pair & 0xffffu;
          if (scale < kScaleInf) top = max(top, scale);
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (top > vlim) {
          const uint32_t bits = max(top << 16, __float_as_uint(kScaleLeast));
          const uint32_t e = bits >> 23;  // the scale lies in [2^(e - 127), 2^(e - 126))
          const float next = copysignf(__uint_as_float((254u + 96u - e) << 23), vmul);  // 2^96 / 2^(e - 127)
          grow = next / vmul;
          vmul = next;
          vlim = min((e << 7) + kScaleRoom, kScaleInf - 1);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(x[nt][i], x[nt][i + 2]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
          const float mn = fmaxf(m[nt][i], mx), a = ex2((m[nt][i] - mn) * sc[nt][i]);
          m[nt][i] = mn;
          mt_[nt][i] = __fadd_rd(mn, kSlack / sc[nt][i]);
          l[nt][i] *= a;
          om[nt][i][0] *= a;
          om[nt][i][1] *= a;
          const float ao = a * grow;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            o[mt][nt][i] *= ao;
            o[mt][nt][i + 2] *= ao;
          }
        }
    };

    // Adds the tile in stage `st` with scores x. Tokens from `valid` on get no weight and, whatever their
    // value pairs hold, count as zeros.
    auto add_tile = [&](uint32_t st, float (*x)[4]) {
      const uint8_t* tile = ring + st * kInt4TileBytes;
      const int valid = wk.tokens[st];
      uint2 vp0 = lds64(tile + kInt4ValuePairs + grp * 8), vp1 = lds64(tile + kInt4ValuePairs + 64 + grp * 8);
      if (valid < kBlockTokens) {
        const bool in0 = grp < valid, in1 = grp + 8 < valid;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (!in0) x[nt][0] = x[nt][1] = -INFINITY;
          if (!in1) x[nt][2] = x[nt][3] = -INFINITY;
        }
        if (!in0) vp0 = make_uint2(0u, 0u);
        if (!in1) vp1 = make_uint2(0u, 0u);
      }
      bool over = false;
      if constexpr (!std::is_same<T, __half>::value)  // scales are not negative: their bits are in their order, NaN above all
        over = (__vmaxu2(__vmaxu2(vp0.x, vp0.y), __vmaxu2(vp1.x, vp1.y)) & 0xffffu) > vlim;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) over = over || fmaxf(x[nt][i], x[nt][i + 2]) > mt_[nt][i];
      if (__any_sync(0xffffffffu, over)) make_room(x, vp0, vp1);

      const uint8_t* vcodes = tile + kInt4ValueCodes + quad * 128 + grp * 16;
      const uint4 vc0 = lds128(vcodes), vc1 = lds128(vcodes + 512);

      // P, its sums, and P * scale of each group, turned around in registers. The maximum is taken off before
      // the product with the scale: of the largest score exactly 0 remains, whatever its size.
      uint32_t pv[2][NT][2][2];  // [group][column tile][tokens 0..7, 8..15][part]
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float2 f0 = unpack2<T>(g == 0 ? vp0.x : vp0.y), f1 = unpack2<T>(g == 0 ? vp1.x : vp1.y);
        const float b0 = fmaf(code0, f0.x, f0.y), b1 = fmaf(code0, f1.x, f1.y);
        const float s0 = f0.x * vmul, s1 = f1.x * vmul;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float* p_ = x[nt];
          if (g == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) p_[i] = ex2((p_[i] - m[nt][i & 1]) * sc[nt][i & 1]);
            l[nt][0] += p_[0] + p_[2];
            l[nt][1] += p_[1] + p_[3];
          }
          om[nt][0][g] = fmaf(p_[0], b0, fmaf(p_[2], b1, om[nt][0][g]));
          om[nt][1][g] = fmaf(p_[1], b0, fmaf(p_[3], b1, om[nt][1][g]));
          split2(p_[0] * s0, p_[1] * s0, pv[g][nt][0][0], pv[g][nt][0][1]);
          split2(p_[2] * s1, p_[3] * s1, pv[g][nt][1][0], pv[g][nt][1][1]);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            pv[g][nt][0][part] = transpose_free(pv[g][nt][0][part]);
            pv[g][nt][1][part] = transpose_free(pv[g][nt][1][part]);
          }
        }
      }

      // O^T: row grp of tile mt is dim 64 (mt / 4) + 8 grp + 2 (mt % 4), row grp + 8 the next dim.
      const uint32_t vw0[4] = {vc0.x, vc0.y, vc0.z, vc0.w}, vw1[4] = {vc1.x, vc1.y, vc1.z, vc1.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t lo[4], hi[4];
        code_pairs_bf16<true>(vw0[w], lo);
        code_pairs_bf16<true>(vw1[w], hi);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t a[4] = {lo[2 * j], lo[2 * j + 1], hi[2 * j], hi[2 * j + 1]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int part = 0; part < 2; ++part)
              mma_free<__nv_bfloat16>(o[2 * w + j][nt], a, pv[w >> 1][nt][0][part], pv[w >> 1][nt][1][part]);
        }
      }
    };

    float x[NT][4];
    for (int k = 0; k < n; ++k) {
      wait(&wk.full[st_con], ph_con);
      if (lost) break;
      scores(st_con, x);
      add_tile(st_con, x);
      // Every lane's reads of the stage have fed its products.
      __syncwarp();
      if (lane == 0) mbar_arrive(&wk.empty[st_con]);
      if (++st_con == kSt) {
        st_con = 0;
        ph_con ^= 1;
      }
    }
    if (lost) break;

    // ---- unit result: sums over the tokens of all rows, then 8 consecutive dims a group and lane ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], off);
          om[nt][i][0] += __shfl_xor_sync(0xffffffffu, om[nt][i][0], off);
          om[nt][i][1] += __shfl_xor_sync(0xffffffffu, om[nt][i][1], off);
        }
    // 2^63 / |vmul|; with 2^70 and 2^66 the units of the codes and that, in two steps within fp32's range.
    const float unit_o = __uint_as_float((317u << 23) - __float_as_uint(fabsf(vmul)));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int head = nt * 8 + 2 * quad + i;
        if (head >= G) continue;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          float y[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            y[2 * j] = fmaf(o[4 * g + j][nt][i] * 0x1p70f, unit_o, om[nt][i][g]);
            y[2 * j + 1] = fmaf(o[4 * g + j][nt][i + 2] * 0x1p66f, unit_o, om[nt][i][g]);
          }
          if (slot < 0) {
            const float inv = l[nt][i] == 0.f ? 0.f : __frcp_rn(l[nt][i]);
            T* dst = out + static_cast<int64_t>(b) * p.out_stride + (static_cast<int64_t>(h) * G + head) * kHeadDim + 64 * g +
                     8 * grp;
            if (aligned(dst, 16)) {
              *reinterpret_cast<uint4*>(dst) =
                  make_uint4(pack2<T>(y[0] * inv, y[1] * inv), pack2<T>(y[2] * inv, y[3] * inv),
                             pack2<T>(y[4] * inv, y[5] * inv), pack2<T>(y[6] * inv, y[7] * inv));
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) dst[j] = from_float<T>(y[j] * inv);
            }
          } else {
            float4* po = reinterpret_cast<float4*>(p.ws.part_o + (static_cast<int64_t>(slot) * G + head) * kHeadDim + 64 * g +
                                                   8 * grp);
            po[0] = make_float4(y[0], y[1], y[2], y[3]);
            po[1] = make_float4(y[4], y[5], y[6], y[7]);
          }
        }
        if (slot >= 0 && grp == 0)  // a finite maximum of a piece without tokens too
          p.ws.part_ml[static_cast<int64_t>(slot) * G + head] = make_float2(fmaxf(m[nt][i] * sc[nt][i], kNoMax), l[nt][i]);
      }
  }

  // Publication and split merge, as in decode_attn_kernel.
  const int planned_warps = __shfl_sync(0xffffffffu, mr.x, 1);
  const int n_entries = min(max(__shfl_sync(0xffffffffu, mr.x, 2), 0), p.num_pairs);
  const int stamp = static_cast<int>(static_cast<unsigned>(__shfl_sync(0xffffffffu, mr.x, 3)) + 1u);  // this launch's
  const int4 share = shfl4(mr, 0);
  int entry = share.x, k = share.y;
  const bool share_ok = planned_warps == total_warps && share.z >= 0 && entry >= 0 && entry <= n_entries;
  const int4 none = make_int4(-1, 0, (1 | (1 << 8)) << 16, 0);
  int4 me = (share_ok && share.z > 0 && entry < n_entries) ? p.ws.split_pairs[entry] : none;
  __syncwarp();
  if (lane == 0) {
    st_release_gpu(&p.ws.warp_flag[gw * kFlagStride], stamp);
    // The CTA's last worker to publish stamps the CTA's flag for all of them.
    if (atom_add_acq_rel_cta(done, 1) == kW - 1)
      st_release_gpu(&p.ws.warp_flag[(total_warps + static_cast<int>(blockIdx.x)) * kFlagStride], stamp);
  }
  int ready_entry = -1;
  if (share_ok) {
    for (int left = share.z; left > 0; --left) {
      if (k >= merge_items(me.z >> 16, G)) {
        ++entry;
        k = 0;
        me = entry < n_entries ? p.ws.split_pairs[entry] : none;
      }
      if (!entry_ok(me, p, total_warps) || k < 0) {
        if (lane == 0) atomicOr(&g_deverr_attn, AEG_DEVERR_PLAN_MISMATCH);
        break;
      }
      if (ready_entry != entry) {
        const int w0 = me.w & 0xffff, nw = me.w >> 16;
        // A worker's flag for each of up to 32 pieces; more of them (a pair of 65,536 tokens has 200) wait
        // for their CTAs' flags, 32 at a time (asking for 200 workers' flags at once delayed the stamps
        // themselves, 32 at a time cost 7 round trips).
        const bool by_cta = nw > 32;
        const int f0 = by_cta ? total_warps + w0 / kW : w0;
        const int nf = by_cta ? (w0 + nw - 1) / kW - w0 / kW + 1 : nw;
        int ok = 1;
        for (int i = 0; i < nf && ok; i += 32) {
          const int f = f0 + i + lane;
          ok = __all_sync(0xffffffffu, i + lane >= nf || f == gw || flag_wait(&p.ws.warp_flag[f * kFlagStride], stamp));
        }
        __syncwarp();
        if (!ok) {
          if (lane == 0) atomicOr(&g_deverr_attn, AEG_DEVERR_WAIT_TIMEOUT);
          break;
        }
        ready_entry = entry;
      }
      merge_item<T, SL::kMergeLoads, true>(p, me, k, lane);
      ++k;
    }
  } else if (lane == 0) {
    atomicOr(&g_deverr_attn, AEG_DEVERR_PLAN_MISMATCH);
  }
}
