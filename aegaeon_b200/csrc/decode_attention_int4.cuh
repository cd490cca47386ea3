// Paged decode attention over a 4-bit KV cache. Part of decode_attention.cu (included there, inside
// its namespace): the plan, the workspace, the split merge and the order of launches are those of
// the 16-bit kernel; what differs is how a worker warp fetches and computes a tile.
//
//   * A (block, head) tile of keys, values and pairs (int4_tile.cuh) is 2304 contiguous bytes: one
//     untiled bulk copy a tile, kStages of them ahead of the compute in each warp's ring. Without a
//     tensor map there is no zero fill, so a tile whose block id is outside the pool is not fetched
//     (its barrier completes at once) and not computed.
//   * No element is dequantised. With K = s c + m per (token, group) and c a whole number 0..15,
//       q . K = sum over groups of  s (q . c) + m (sum of q)
//       sum_t p_t V_t = sum_t (p_t s_t) c_t + sum_t p_t m_t
//     so the codes go to the tensor cores as they are, exactly, and scales and minima meet them
//     in fp32. A code becomes a 16-bit float with one AND-OR: a nibble under the exponent of a power
//     of two B reads as B + c, and the constant is taken out with the minima (m - B s in place of
//     m), in fp32. B is 64 or 128 for the keys, where it is out again after four MMAs, and 16 for
//     the values (see the fold below).
//   * S^T = K Q^T as in the 16-bit kernel (16 tokens x 8 heads of the group, m16n8k16), in the
//     query's own type. A lane's codes of a token are one 16-byte load; which dim sits where in the
//     contraction is free as long as the query fragments follow.
//   * O^T += V^T P^T with codes and P * s as fp16, P * s brought to within 2^15 by a power of two that
//     follows the largest scale the warp has met: 11 bits for everything down to 2^-23 of the
//     largest product (bf16 would keep 8 and need a second MMA for the rest). Token pairs share a
//     32-bit word, so that the transposed fragment comes out of the same AND-OR without a
//     transposing load. sum p m is 4 FMAs a token and lane.
//   * The tensor cores cut off what an addition pushes out of the accumulator, always downwards, so
//     a sum that carries 16 sum(p s) along drifts with its length (at B = 128 the error of 4096
//     tokens was 2.5 times that of the output's own rounding). Every kFold tiles the constant's
//     share is therefore taken out of O, which leaves sums of the size of the result.
//   * The running maximum moves only when a score exceeds it by kSlack (log2 units): sums are fp32, and
//     most tiles need one vote instead of a reduction over the tokens and a rescaling of O.
//   * Tiles are requested several at a time, one lane each, so that walking the units and the block
//     table costs a fraction of an instruction stream a tile.
//
// What bounds it: at 4.5 bits an element the work per byte is 3.6 times that of the 16-bit kernel,
// so issue slots count as much as bytes.

template <int NT>
struct Int4Smem {
  // More worker warps than the 16-bit kernel's 8 hide the latency of a tile's longer chain, as far
  // as the registers of one CTA per SM go.
  static constexpr int kWarps = NT == 1 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kStages = NT == 1 ? 7 : 10;
  static constexpr int kBatch = kStages / 2;  // free stages at which a warp requests more
  static constexpr int kMergeLoads = NT == 1 ? 8 : kMergeBatch;  // pieces of a merge in flight per lane
  static constexpr int kQSlot = 8 * NT * kHeadDim * 2;
  static constexpr int kPerWarp = kStages * kInt4TileBytes + kQSlot;
  static constexpr int kOffBars = kWarps * kPerWarp;
  static constexpr int kBarsPerWarp = kStages + 2;  // stages, query slot, one scratch word
  static constexpr int kTotal = kOffBars + kWarps * kBarsPerWarp * 8;
  static constexpr size_t kDynamic = size_t(kTotal) + 128;  // + alignment slack
  static_assert(kPerWarp % 128 == 0 && kDynamic <= 232448, "ring alignment and capacity");
};

// (x & mask) | bits in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
  return r;
}
// Nibbles k and k + 4 (k = 0..3) of a key word as two elements of T, code + kKeyBias<T>.
template <typename T>
__device__ __forceinline__ uint32_t key_pair(uint32_t w, int k);
template <>
__device__ __forceinline__ uint32_t key_pair<__half>(uint32_t w, int k) {
  return and_or(k == 0 ? w << 4 : w >> (4 * (k - 1)), 0x00f000f0u, 0x54005400u);
}
template <>
__device__ __forceinline__ uint32_t key_pair<__nv_bfloat16>(uint32_t w, int k) {
  return and_or(w >> (4 * k), 0x000f000fu, 0x43004300u);
}
template <typename T>
constexpr float kKeyBias = std::is_same<T, __half>::value ? 64.f : 128.f;

// The same of a value word, as fp16 and with a bias of 16.
__device__ __forceinline__ uint32_t value_pair(uint32_t w, int k) {
  return and_or(k < 2 ? w << (6 - 4 * k) : w >> (4 * k - 6), 0x03c003c0u, 0x4c004c00u);
}
constexpr float kValueBias = 16.f;
// Bits of a scale: infinity, and the mantissa.
template <typename T>
constexpr uint32_t kScaleInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
template <typename T>
constexpr uint32_t kScaleMantissa = std::is_same<T, __half>::value ? 0x3ffu : 0x7fu;
constexpr float kValueMiddle = 8.f;

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(addr));
  return r;
}
__device__ __forceinline__ void bulk_load_1d_hint(void* smem_dst, const void* gmem_src, uint32_t bytes, uint64_t* bar,
                                                  uint64_t l2_policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(gmem_src)), "r"(bytes), "r"(smem_u32(bar)), "l"(l2_policy)
      : "memory");
}

template <typename T, int NT>
__global__ void __launch_bounds__(Int4Smem<NT>::kThreads, 1) decode_attn_int4_kernel(const AttnParams p) {
  using SL = Int4Smem<NT>;
  constexpr int kW = SL::kWarps, kSt = SL::kStages, kBatch = SL::kBatch;
  constexpr float kNoMax = -1e30f;     // the running maximum before the first score
  constexpr float kSlack = 6.f;        // scores may exceed the running maximum by this (log2 units)
  constexpr float kTop = 512.f;        // largest scaled scale: 2^9 * 2^kSlack = 2^15 fits fp16
  constexpr int kFold = 32;            // tiles between two removals of the constant from O
  const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 127) & ~127u) - raw);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * SL::kPerWarp;
  T* qslot = reinterpret_cast<T*>(ring + kSt * kInt4TileBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SL::kOffBars) + warp * SL::kBarsPerWarp;
  uint64_t* qbar = full + kSt;
  uint32_t* qdep_slot = reinterpret_cast<uint32_t*>(full + kSt + 1);

  if (lane == 0) {
    for (int s = 0; s < kSt; ++s) mbar_init(&full[s], 1);
    mbar_init(qbar, 1);
    fence_mbar_init();
  }
  __syncwarp();

  // Plan records, as in decode_attn_kernel.
  const int gw = static_cast<int>(blockIdx.x) * kW + warp;
  const uint64_t keep = l2_policy_evict_last();
  int4 r0 = make_int4(0, 0, 0, 0);
  auto load_plan = [&]() {
    if (lane < 3)
      r0 = ld_hint(&p.ws.warp_rec[3 * gw + lane], keep);
    else if (lane == 3)
      r0.x = ld_hint(&p.ws.warp_rec[3 * (gw + 1)].x, keep);
    else if (lane == 4)
      r0.x = ld_hint(&p.ws.header[kHdrWarps], keep);
    else if (lane == 5)
      r0.x = ld_hint(&p.ws.header[kHdrUnits], keep);
    else if (lane == 6)
      r0.x = ld_hint(&p.ws.header[kHdrSplitPairs], keep);
    else if (lane == 7)
      r0 = ld_hint(&p.ws.merge_rec[gw], keep);
  };
  if (p.plan_ready) load_plan();
  const bool early = p.plan_ready && p.prefetch_kv;
  if (!early) {
    pdl_wait_primary();
    pdl_launch_dependents();
    if (!p.plan_ready) load_plan();
  }

  const int G = p.G;
  const int Hkv = p.Hkv;
  const int total_warps = static_cast<int>(gridDim.x) * kW;
  const uint64_t pol = l2_policy_evict_first();
  const T* q = static_cast<const T*>(p.q);
  T* out = static_cast<T*>(p.out);
  const int quad = lane & 3;  // column pair of the accumulator fragment
  const int grp = lane >> 2;  // row of the accumulator fragment

  bool abort = false;
  uint32_t g_iss = 0, g_con = 0;      // tiles requested / consumed by this warp
  uint32_t st_iss = 0, st_con = 0;    // their stages
  uint32_t ph_con = 0;
  const float sc = fmaxf(fabsf(p.scale_log2), 1e-30f);  // not 0, so that -infinity stays below all scores
  const float slack = kSlack / sc;
  uint32_t bad = 0;                   // stages whose block id was outside the pool
  uint32_t q_phase = 0;

  auto report_timeout = [&]() {
    abort = true;
    if (lane == 0) atomicOr(&g_deverr_attn, AEG_DEVERR_WAIT_TIMEOUT);
  };

  const int u_beg = __shfl_sync(0xffffffffu, r0.x, 0);
  const int u_end = __shfl_sync(0xffffffffu, r0.x, 3);
  const int planned_warps = __shfl_sync(0xffffffffu, r0.x, 4);
  const int planned_units = __shfl_sync(0xffffffffu, r0.x, 5);
  const int n_entries = min(max(__shfl_sync(0xffffffffu, r0.x, 6), 0), p.num_pairs);
  const int4 mr = shfl4(r0, 7);
  int n_units = u_end - u_beg;
  if (!(planned_warps == total_warps && planned_units <= p.max_units && u_beg >= 0 && u_beg <= u_end &&
        u_end <= planned_units)) {
    if (lane == 0 && n_units != 0) atomicOr(&g_deverr_attn, AEG_DEVERR_PLAN_MISMATCH);
    n_units = 0;
  }

  // Unit records, one per lane: lane (k % 32) holds the worker's unit k for the 32 units from the
  // one being computed on. Lane 0 takes unit 0 from the start record.
  int4 ra = shfl4(r0, 1), rb = shfl4(r0, 2);
  if (lane > 0) {
    if (lane < n_units) {
      ra = ld_hint(&p.ws.units[2 * (u_beg + lane)], keep);
      rb = ld_hint(&p.ws.units[2 * (u_beg + lane) + 1], keep);
    } else {
      ra = make_int4(0, 0, 0, -1);
      rb = make_int4(0, 0, 0, 0);
    }
  }

  auto load_q = [&](int k) {
    const int4 a = shfl4(ra, k & 31), bb = shfl4(rb, k & 31);
    if (unit_items(a, bb, p) == 0) {
      if (lane == 0) mbar_arrive(qbar);
      return;
    }
    const int b = a.x / Hkv, h = a.x % Hkv;
    const T* qsrc = q + static_cast<int64_t>(b) * p.q_stride + static_cast<int64_t>(h) * G * kHeadDim;
    const uint32_t qbytes = G * kHeadDim * 2;
    if (p.q_bulk) {
      if (lane == 0) {
        mbar_arrive_expect_tx(qbar, qbytes);
        bulk_load_1d(qslot, qsrc, qbytes, qbar);
      }
    } else {
      for (int i = lane; i < G * kHeadDim / 2; i += 32)
        reinterpret_cast<uint32_t*>(qslot)[i] = reinterpret_cast<const uint32_t*>(qsrc)[i];
      __syncwarp();
      if (lane == 0) mbar_arrive(qbar);
    }
  };

  // Issue walker: requests the worker's tiles in order, one lane a tile. Block ids of items 0..2 of
  // a unit come with its record (lanes 0..2), later ones from a 32-entry chunk of the block table
  // loaded when the walker enters the unit (the chunk after it one chunk ahead).
  int ik = -1, ii = 0, in_ = 0, irec = 0, itbase = 3, itbl = 0, itnext = 0;
  const int* itab = p.tables;
  const T* ihead = static_cast<const T*>(p.k_cache);
  auto issue_enter = [&](int k) {
    ik = k;
    ii = 0;
    in_ = 0;
    if (k >= n_units) return;
    const int4 a = shfl4(ra, k & 31), bb = shfl4(rb, k & 31);
    in_ = unit_items(a, bb, p);
    if (in_ == 0) return;
    ihead = static_cast<const T*>(p.k_cache) + static_cast<int64_t>(a.x % Hkv) * kInt4TileElems;
    irec = lane == 0 ? bb.y : (lane == 1 ? bb.z : bb.w);
    itab = p.tables + static_cast<int64_t>(a.x / Hkv) * p.table_stride + a.y;
    itbase = 3;
    itbl = lane < in_ - 3 ? itab[3 + lane] : 0;
    itnext = lane < in_ - 35 ? itab[35 + lane] : 0;
  };
  auto refill = [&]() {
    int room = kSt - static_cast<int>(g_iss - g_con);
    while (room > 0) {
      if (ii >= in_) {
        if (ik >= n_units) break;
        issue_enter(ik + 1);
        continue;
      }
      int first, left, blk;
      const bool from_rec = ii < 3;
      if (from_rec) {
        first = ii;
        left = min(in_, 3) - ii;
        blk = irec;
      } else {
        if (ii - itbase >= 32) {
          itbase += 32;
          itbl = itnext;
          itnext = lane < in_ - itbase - 32 ? itab[itbase + 32 + lane] : 0;
        }
        first = ii - itbase;
        left = min(in_, itbase + 32) - ii;
        blk = itbl;
      }
      const int cnt = min(left, room);
      const int r = lane - first;  // this lane's tile of the batch
      const bool mine = r >= 0 && r < cnt;
      const bool inside = static_cast<uint32_t>(blk) < static_cast<uint32_t>(p.num_blocks);
      uint32_t st = st_iss + static_cast<uint32_t>(r);
      st = st >= kSt ? st - kSt : st;
      if (mine && !abort) {
        if (inside) {
          mbar_arrive_expect_tx(&full[st], kInt4TileBytes);
          bulk_load_1d_hint(ring + st * kInt4TileBytes, ihead + static_cast<int64_t>(blk) * p.block_stride, kInt4TileBytes,
                            &full[st], pol);
        } else {
          atomicOr(&g_deverr_attn, AEG_DEVERR_BLOCK_ID_RANGE);
          mbar_arrive(&full[st]);
        }
      }
      const uint32_t out_of_pool = __ballot_sync(0xffffffffu, mine && !inside);
      if (out_of_pool | bad) {
        for (int j = 0; j < cnt; ++j) {
          const uint32_t sj = (st_iss + j) % kSt;
          bad = (bad & ~(1u << sj)) | (((out_of_pool >> (first + j)) & 1u) << sj);
        }
      }
      g_iss += cnt;
      st_iss = st_iss + cnt >= kSt ? st_iss + cnt - kSt : st_iss + cnt;
      ii += cnt;
      // The chunk requested on entering the unit may still be on its way: later items wait for the
      // next call, unless nothing else is in the ring.
      room = from_rec && g_iss - g_con >= 3 ? 0 : room - cnt;
    }
  };

  if (early) {
    refill();
    pdl_wait_primary();
    pdl_launch_dependents();
  }
  if (n_units > 0) load_q(0);
  refill();
  const int epoch_word = lane == 0 ? ld_relaxed_gpu(&p.ws.warp_flag[gw * kFlagStride]) : 0;

  for (int c = 0; c < n_units; ++c) {
    if (c > 0 && lane == ((c - 1) & 31) && c + 31 < n_units) {
      ra = p.ws.units[2 * (u_beg + c + 31)];
      rb = p.ws.units[2 * (u_beg + c + 31) + 1];
    }
    const int4 ua = shfl4(ra, c & 31), ub = shfl4(rb, c & 31);
    const int n = unit_items(ua, ub, p);
    if (n == 0 && lane == 0) atomicOr(&g_deverr_attn, AEG_DEVERR_PLAN_MISMATCH);
    const int b = ua.x / Hkv, h = ua.x % Hkv, j0 = ua.y, slot = ua.w, n_ctx = ub.x;

    if (!abort && !mbar_wait_bounded(qbar, q_phase, kWaitLimitNs)) report_timeout();
    q_phase ^= 1;
    // Query fragments: contraction step 2 w + u pairs dims (d, d + 4) and (d + 1, d + 5) with
    // d = 32 w + 8 quad + 2 u, as the code words do. Then the sums of q over each group, for the
    // fragment's two columns.
    // A negative scale goes into the sign of q, so that larger sums always mean larger scores.
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    uint32_t qf[NT][8][2];
    float qs[NT][2][2];  // [column][group]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + grp;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (head < G) x = lds128(smem_u32(qslot) + head * (kHeadDim * 2) + w * 64 + quad * 16);
        x = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
        qf[nt][2 * w][0] = __byte_perm(x.x, x.z, 0x5410);
        qf[nt][2 * w][1] = __byte_perm(x.x, x.z, 0x7632);
        qf[nt][2 * w + 1][0] = __byte_perm(x.y, x.w, 0x5410);
        qf[nt][2 * w + 1][1] = __byte_perm(x.y, x.w, 0x7632);
        const float2 f0 = unpack2<T>(x.x), f1 = unpack2<T>(x.y), f2 = unpack2<T>(x.z), f3 = unpack2<T>(x.w);
        sum[w >> 1] += ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        qs[nt][0][g] = __shfl_sync(0xffffffffu, sum[g], 8 * quad);
        qs[nt][1][g] = __shfl_sync(0xffffffffu, sum[g], 8 * quad + 4);
      }
    }
    // The next unit's rows overwrite the slot: make every lane's slot reads complete first.
    {
      uint32_t dep = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) dep ^= qf[nt][ks][0] ^ qf[nt][ks][1];
      if (lane == 0) *qdep_slot = dep;
    }
    __syncwarp();
    if (c + 1 < n_units) load_q(c + 1);
    if (n == 0) continue;

    // Running maximum of the unscaled scores, that times the scale, and the score from which it moves;
    // sum of p; sum of p * (minimum + middle * scale) [column][group]; sum of the rounded P * scale
    // [group]. O and the last are held times `vmul`.
    float o[8][NT][4];
    float m[NT][2], ms[NT][2], mt_[NT][2], l[NT][2], om[NT][2][2], ps[2][NT][4];
    float vmul = kTop;
    uint32_t vlim = 0;  // bits of the largest scale allowed for
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[nt][i] = kNoMax;
        ms[nt][i] = kNoMax * sc;
        mt_[nt][i] = kNoMax + slack;
        l[nt][i] = om[nt][i][0] = om[nt][i][1] = 0.f;
        ps[i][nt][0] = ps[i][nt][1] = ps[i][nt][2] = ps[i][nt][3] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.f;
    }
    // Takes the codes' constant out of O.
    auto fold = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
          for (int mt = 4 * g; mt < 4 * g + 4; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[mt][nt][i] = fmaf(-(kValueBias + kValueMiddle), ps[g][nt][i], o[mt][nt][i]);
          ps[g][nt][0] = ps[g][nt][1] = ps[g][nt][2] = ps[g][nt][3] = 0.f;
        }
    };

    // Scores of the tile in stage `st`, unscaled: S^T, one accumulator per group; rows are tokens grp
    // and grp + 8.
    auto scores = [&](uint32_t st, float (&x)[NT][4]) {
      const uint32_t tile = smem_u32(ring) + st * kInt4TileBytes;
      const uint4 kc0 = lds128(tile + grp * 64 + quad * 16), kc1 = lds128(tile + 512 + grp * 64 + quad * 16);
      const uint2 kp0 = lds64(tile + kInt4KeyPairs + grp * 8), kp1 = lds64(tile + kInt4KeyPairs + 64 + grp * 8);
      const uint32_t kw0[4] = {kc0.x, kc0.y, kc0.z, kc0.w}, kw1[4] = {kc1.x, kc1.y, kc1.z, kc1.w};
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int w = 2 * g; w < 2 * g + 2; ++w)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t a[4] = {key_pair<T>(kw0[w], 2 * u), key_pair<T>(kw1[w], 2 * u), key_pair<T>(kw0[w], 2 * u + 1),
                                   key_pair<T>(kw1[w], 2 * u + 1)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) MmaF32<T>::run(s[nt], a, qf[nt][2 * w + u][0], qf[nt][2 * w + u][1]);
          }
        const float2 f0 = unpack2<T>(g == 0 ? kp0.x : kp0.y), f1 = unpack2<T>(g == 0 ? kp1.x : kp1.y);
        const float b0 = fmaf(-kKeyBias<T>, f0.x, f0.y), b1 = fmaf(-kKeyBias<T>, f1.x, f1.y);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x[nt][i] = fmaf(f0.x, s[nt][i], g == 0 ? b0 * qs[nt][i][g] : fmaf(b0, qs[nt][i][g], x[nt][i]));
            x[nt][i + 2] = fmaf(f1.x, s[nt][i + 2], g == 0 ? b1 * qs[nt][i][g] : fmaf(b1, qs[nt][i][g], x[nt][i + 2]));
          }
      }
    };

    // Makes room for the scores x and the scales under vtop: the maxima move to the tile's, and what
    // was summed so far follows.
    auto make_room = [&](const float (&x)[NT][4], uint32_t vtop) {
      uint32_t top = vtop;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
      float grow = 1.f;
      if (top > vlim && top < kScaleInf<T>) {
        // The power of two above the scale, kept in range for the tiniest ones. NaN needs no room: it
        // makes the result NaN by itself.
        const float t = fmaxf(unpack2<T>(top).x, 6.103515625e-05f);
        const uint32_t e = __float_as_uint(t) >> 23;  // t in [2^(e - 127), 2^(e - 126))
        const float next = __uint_as_float((253u - e) << 23) * kTop;
        grow = vlim == 0 ? 1.f : next / vmul;  // nothing but zeros was added before the first scale
        vmul = next;
        vlim = bits16(from_float<T>(t)) | kScaleMantissa<T>;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(x[nt][i], x[nt][i + 2]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
          const float mn = fmaxf(m[nt][i], mx), a = ex2((m[nt][i] - mn) * sc);
          m[nt][i] = mn;
          ms[nt][i] = mn * sc;
          mt_[nt][i] = mn + slack;
          l[nt][i] *= a;
          om[nt][i][0] *= a;
          om[nt][i][1] *= a;
          const float ao = a * grow;
          ps[0][nt][i] *= ao;
          ps[0][nt][i + 2] *= ao;
          ps[1][nt][i] *= ao;
          ps[1][nt][i + 2] *= ao;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            o[mt][nt][i] *= ao;
            o[mt][nt][i + 2] *= ao;
          }
        }
    };

    // Adds the tile in stage `st` with scores x. Tokens from nvalid on get no weight and, whatever their
    // value pairs hold, count as zeros. With kNext the next tile's scores are made on the way: their
    // chain of MMAs runs beside this tile's exponents and products.
    auto add_tile = [&](auto next_tag, uint32_t st, uint32_t st_next, float (&x)[NT][4], float (&x_next)[NT][4], int nvalid) {
      constexpr bool kNext = decltype(next_tag)::value;
      const uint32_t tile = smem_u32(ring) + st * kInt4TileBytes;
      uint2 vp0 = lds64(tile + kInt4ValuePairs + grp * 8), vp1 = lds64(tile + kInt4ValuePairs + 64 + grp * 8);
      if (!kNext && nvalid < kBlockTokens) {  // only a sequence's last tile is partly filled
        const bool in0 = grp < nvalid, in1 = grp + 8 < nvalid;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (!in0) x[nt][0] = x[nt][1] = -INFINITY;
          if (!in1) x[nt][2] = x[nt][3] = -INFINITY;
        }
        if (!in0) vp0 = make_uint2(0u, 0u);
        if (!in1) vp1 = make_uint2(0u, 0u);
      }
      // Scales are not negative, so their bits are in their order; NaN is above all.
      const uint32_t vtop = __vmaxu2(__vmaxu2(vp0.x, vp0.y), __vmaxu2(vp1.x, vp1.y)) & 0xffffu;
      bool over = vtop > vlim;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        over = over || fmaxf(x[nt][0], x[nt][2]) > mt_[nt][0] || fmaxf(x[nt][1], x[nt][3]) > mt_[nt][1];
      if (__any_sync(0xffffffffu, over)) make_room(x, vtop);

      if constexpr (kNext) scores(st_next, x_next);
      const uint4 vc0 = lds128(tile + kInt4ValueCodes + quad * 128 + grp * 16);
      const uint4 vc1 = lds128(tile + kInt4ValueCodes + 512 + quad * 128 + grp * 16);

      // P, its sums, and P * scale of each group, turned around in registers.
      uint32_t pv[2][NT][2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float2 f0 = unpack2<T>(g == 0 ? vp0.x : vp0.y), f1 = unpack2<T>(g == 0 ? vp1.x : vp1.y);
        const float b0 = fmaf(kValueMiddle, f0.x, f0.y), b1 = fmaf(kValueMiddle, f1.x, f1.y);
        const float s0 = f0.x * vmul, s1 = f1.x * vmul;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (g == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[nt][i] = ex2(fmaf(x[nt][i], sc, -ms[nt][i & 1]));
            l[nt][0] += x[nt][0] + x[nt][2];
            l[nt][1] += x[nt][1] + x[nt][3];
          }
          om[nt][0][g] = fmaf(x[nt][0], b0, fmaf(x[nt][2], b1, om[nt][0][g]));
          om[nt][1][g] = fmaf(x[nt][1], b0, fmaf(x[nt][3], b1, om[nt][1][g]));
          pv[g][nt][0] = movmatrix_trans(pack2<__half>(x[nt][0] * s0, x[nt][1] * s0));
          pv[g][nt][1] = movmatrix_trans(pack2<__half>(x[nt][2] * s1, x[nt][3] * s1));
          MmaF32<__half>::run(ps[g][nt], ones, pv[g][nt][0], pv[g][nt][1]);
        }
      }

      // O^T: row grp of tile mt is dim 64 (mt / 4) + 8 grp + 2 (mt % 4), row grp + 8 the next dim.
      const uint32_t vw0[4] = {vc0.x, vc0.y, vc0.z, vc0.w}, vw1[4] = {vc1.x, vc1.y, vc1.z, vc1.w};
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        const int w = mt >> 1, u = 2 * (mt & 1);
        const uint32_t a[4] = {value_pair(vw0[w], u), value_pair(vw0[w], u + 1), value_pair(vw1[w], u),
                               value_pair(vw1[w], u + 1)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) MmaF32<__half>::run(o[mt][nt], a, pv[mt >> 2][nt][0], pv[mt >> 2][nt][1]);
      }
    };

    // The unit's tiles. A tile that is not computed (an id outside the pool) breaks the chain of scores
    // made ahead.
    float x[NT][4], x_next[NT][4];
    bool have = false;  // x holds the scores of the tile in stage st_con, which has landed
    for (int k = 0; k < n; ++k) {
      if (!have && !abort && !mbar_wait_bounded(&full[st_con], ph_con, kWaitLimitNs)) report_timeout();
      const uint32_t st_next = st_con + 1 == kSt ? 0 : st_con + 1;
      const uint32_t ph_next = st_con + 1 == kSt ? ph_con ^ 1 : ph_con;
      const int nvalid = min(kBlockTokens, n_ctx - (j0 + k) * kBlockTokens);
      const bool use = !abort && nvalid > 0 && !((bad >> st_con) & 1u);
      if (use && !have) scores(st_con, x);
      have = false;
      if (k + 1 < n && use && !((bad >> st_next) & 1u)) {
        if (!mbar_wait_bounded(&full[st_next], ph_next, kWaitLimitNs)) {
          report_timeout();
        } else {
          add_tile(std::true_type{}, st_con, st_next, x, x_next, kBlockTokens);
          have = true;
        }
      } else if (use) {
        add_tile(std::false_type{}, st_con, st_next, x, x_next, nvalid);
      }
      if ((k & (kFold - 1)) == kFold - 1) fold();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[nt][i] = x_next[nt][i];
      __syncwarp();
      ++g_con;
      st_con = st_next;
      ph_con = ph_next;
      if (kSt - static_cast<int>(g_iss - g_con) >= kBatch || k + 1 == n) refill();
    }

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
    fold();
    const float unit_o = 1.f / vmul;
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
            y[2 * j] = fmaf(o[4 * g + j][nt][i], unit_o, om[nt][i][g]);
            y[2 * j + 1] = fmaf(o[4 * g + j][nt][i + 2], unit_o, om[nt][i][g]);
          }
          if (slot < 0) {
            const float inv = l[nt][i] > 0.f ? 1.f / l[nt][i] : (l[nt][i] == 0.f ? 0.f : l[nt][i]);
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
        if (slot >= 0 && grp == 0) p.ws.part_ml[static_cast<int64_t>(slot) * G + head] = make_float2(ms[nt][i], l[nt][i]);
      }
  }

  // Publication and split merge, as in decode_attn_kernel.
  int entry = mr.x, k = mr.y;
  const bool share_ok = planned_warps == total_warps && mr.z >= 0 && entry >= 0 && entry <= n_entries;
  const int4 none = make_int4(-1, 0, (1 | (1 << 8)) << 16, 0);
  int4 me = (share_ok && mr.z > 0 && entry < n_entries) ? p.ws.split_pairs[entry] : none;
  const int epoch = __shfl_sync(0xffffffffu, epoch_word, 0);
  const int stamp = static_cast<int>(static_cast<unsigned>(epoch) + 1u);
  __syncwarp();
  if (lane == 0) st_release_gpu(&p.ws.warp_flag[gw * kFlagStride], stamp);
  int ready_entry = -1;
  if (share_ok) {
    for (int left = mr.z; left > 0; --left) {
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
        int ok = 1;
        for (int i = 0; i < nw && ok; i += 32) {
          const int ww = w0 + i + lane;
          ok = __all_sync(0xffffffffu,
                          i + lane >= nw || ww == gw || flag_wait(&p.ws.warp_flag[ww * kFlagStride], stamp));
        }
        __syncwarp();
        if (!ok) {
          if (lane == 0) atomicOr(&g_deverr_attn, AEG_DEVERR_WAIT_TIMEOUT);
          break;
        }
        ready_entry = entry;
      }
      merge_item<T, SL::kMergeLoads>(p, me, k, lane);
      ++k;
    }
  } else if (lane == 0) {
    atomicOr(&g_deverr_attn, AEG_DEVERR_PLAN_MISMATCH);
  }
}
