// Shared KV blocks: forking rows of the block tables over reference counts, freeing them, and
// moving a fragmented pool's live blocks to its lowest ids.
//
// State, all on the device: ref_counts[b] counts the table rows that hold block b (0 = free),
// block_tables and seq_lens are the resident tables of step_inputs.cu. Nothing is read back: the
// blocks to take, to copy and to move are found by the kernels, so a beam step or a compaction costs
// launches, not a synchronisation. Free blocks are always taken lowest id first, in the order of
// the call's entries, so results do not depend on which thread came first.
//
// A fork shares the source row's full blocks (their counts go up) and copies its partly filled last
// block, into which both rows will write. fork_plan_kernel (one CTA) checks the entries, ranks those
// that need a block and finds that many free ones, leaving the scan of the counts at the last one it
// needs; fork_apply_kernel copies the tails, 16-byte vectors grid-stride over (entry, 32 KiB segment)
// as copy_blocks does, and writes the rows. compact_blocks has the same two parts.
//
// Measured: dropping and forking 192 rows whose tails are 28-layer blocks of 917,504 bytes 48 us (the copies
// alone 331 MB, partly from L2), 24 rows of 131,072-byte blocks 9.0 us, of which the one-CTA plan ~4;
// compacting a pool of 2048 such blocks, 470 of them moving, 144 us (5.9 TB/s, 0.90 of the measured copy
// rate); the bookkeeping of 200,000 blocks 140 us.
#include "aeg_common.cuh"

#include <algorithm>

namespace aeg {
namespace {

__device__ unsigned int g_deverr_pool = 0;

constexpr int kBlockTokens = 16;
constexpr int kPlanThreads = 1024;
constexpr int kScanRows = 8;  // rows of 32 counts a warp takes per step of a scan, all loads in flight
constexpr int kScanStep = kPlanThreads * kScanRows;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;
constexpr int64_t kSegVecs = int64_t(kCopyThreads) * kCopyUnroll;  // 32 KiB a segment

__device__ __forceinline__ void report(uint32_t bits) { atomicOr(&g_deverr_pool, bits); }

// Exclusive sum of one value a thread over the CTA; `total` gets the sum. The leading barrier lets
// calls follow one another on the same scratch.
__device__ __forceinline__ int cta_scan(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 31) s_warp[wid] = incl;
  __syncthreads();
  int w = s_warp[lane];  // kPlanThreads / 32 = 32 warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += t;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, max(wid, 1) - 1);
  return (wid > 0 ? before : 0) + incl - v;
}
static_assert(kPlanThreads == 1024, "cta_scan sums 32 warps");

__device__ __forceinline__ int ld_relaxed(const int* p) {
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void st_relaxed(int* p, int v) {
  asm volatile("st.relaxed.gpu.global.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

__device__ __forceinline__ bool valid_id(int64_t id, int64_t n) { return id >= 0 && id < n; }

// The share of CTA-wide work (item) of copying one block: segment `seg` of src -> dst.
template <bool kVec>
__device__ __forceinline__ void copy_segment(const uint8_t* src, uint8_t* dst, int64_t block_bytes, int64_t seg) {
  if constexpr (kVec) {
    const uint4* s = reinterpret_cast<const uint4*>(src);
    uint4* d = reinterpret_cast<uint4*>(dst);
    const int64_t vecs = block_bytes / 16, base = seg * kSegVecs + threadIdx.x;
    if (base + (kCopyUnroll - 1) * kCopyThreads < vecs) {
      uint4 v[kCopyUnroll];
#pragma unroll
      for (int u = 0; u < kCopyUnroll; ++u) v[u] = __ldcs(s + base + u * kCopyThreads);
#pragma unroll
      for (int u = 0; u < kCopyUnroll; ++u) __stcs(d + base + u * kCopyThreads, v[u]);
    } else {
#pragma unroll
      for (int u = 0; u < kCopyUnroll; ++u) {
        const int64_t k = base + u * kCopyThreads;
        if (k < vecs) __stcs(d + k, __ldcs(s + k));
      }
    }
  } else {
    const int64_t begin = seg * kSegVecs * 16;
    const int64_t end = min(begin + kSegVecs * 16, block_bytes);
    for (int64_t k = begin + threadIdx.x; k < end; k += kCopyThreads) dst[k] = src[k];
  }
}

// The counts of a warp's blocks b, b + 32, ... (b includes the lane); -1 past the end, which is neither
// free nor live.
__device__ __forceinline__ void load_counts(const int* ref_counts, int64_t b, int num_blocks, int (&rc)[kScanRows]) {
#pragma unroll
  for (int k = 0; k < kScanRows; ++k) rc[k] = b + 32 * k < num_blocks ? ref_counts[b + 32 * k] : -1;
}

struct PoolParams {
  uint8_t* pool;
  int64_t block_bytes;
  int64_t segs;  // segments of a block
  int num_blocks;
  int* ref_counts;
  int* tables;
  int table_stride;
  int rows;
  int* seq_lens;
};

// Pointers are not __restrict__: a load promised to be invariant may be moved ahead of the grid-dependency
// wait, and the kernel before this one may itself have started early.

// ---- fork --------------------------------------------------------------------------------------

// What fork_plan_kernel leaves for fork_apply_kernel, one per entry: {source row, target row, length
// (-1: refused), id of the copied last block or -1} and the id that block is copied from.
struct ForkScratch {
  int4* entry;
  int* tail;
  int* free_ids;
};

__global__ void __launch_bounds__(kPlanThreads, 1)
fork_plan_kernel(const PoolParams p, const int64_t* src, const int64_t* dst, int n, ForkScratch ws,
                 int* new_blocks) {
  __shared__ int s_warp[32];
  pdl_enter();
  const int tid = threadIdx.x;
  const int cap = p.table_stride * kBlockTokens;
  // Entries in themselves. Lengths are read past the L1 cache: the claims below change them.
  for (int i = tid; i < n; i += kPlanThreads) {
    const int64_t s = src[i], d = dst[i];
    int4 e = make_int4(-1, -1, -1, -1);
    int tail = -1;
    if (valid_id(s, p.rows) && valid_id(d, p.rows)) {
      const int len = __ldcg(&p.seq_lens[s]);
      if (len >= 0 && len <= cap && __ldcg(&p.seq_lens[d]) == 0) {
        e = make_int4(static_cast<int>(s), static_cast<int>(d), len, -1);
        if (len % kBlockTokens) {
          tail = p.tables[s * p.table_stride + len / kBlockTokens];
          if (!valid_id(tail, p.num_blocks)) {
            e.z = -1;
            report(AEG_DEVERR_BLOCK_ID_RANGE);
          } else if (p.ref_counts[tail] <= 0) {  // free: this call may give it out while it is copied
            e.z = -1;
            report(AEG_DEVERR_POOL_ENTRY);
          }
        }
      } else {
        report(AEG_DEVERR_POOL_ENTRY);
      }
    } else {
      report(AEG_DEVERR_POOL_ENTRY);
    }
    ws.entry[i] = e;
    ws.tail[i] = tail;
  }
  __syncthreads();
  // A target row named twice goes to its first entry: each leaves its (negative) place in the empty
  // row's length, and the least stays.
  for (int i = tid; i < n; i += kPlanThreads)
    if (ws.entry[i].z >= 0) atomicMin(&p.seq_lens[ws.entry[i].y], i - n);
  __syncthreads();
  int want = 0;  // blocks wanted so far
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    bool need = false;
    if (i < n && ws.entry[i].z >= 0) {
      if (__ldcg(&p.seq_lens[ws.entry[i].y]) != i - n) {
        ws.entry[i].z = -1;
        report(AEG_DEVERR_POOL_ENTRY);
      } else {
        need = ws.tail[i] >= 0;
      }
    }
    int total;
    const int rank = cta_scan(need ? 1 : 0, s_warp, total);
    if (need) ws.entry[i].w = want + rank;
    want += total;
  }
  // The first `want` free blocks; the next step's counts are on their way while this one's are summed.
  // A warp takes consecutive rows of 32, so that ballots rank them.
  int found = 0;
  const int lane = tid & 31;
  const int64_t first = int64_t(tid >> 5) * 32 * kScanRows + lane;
  int ahead[kScanRows];
  if (want > 0) load_counts(p.ref_counts, first, p.num_blocks, ahead);
  for (int64_t b0 = 0; b0 < p.num_blocks && found < want; b0 += kScanStep) {
    uint32_t is_free[kScanRows];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < kScanRows; ++k) {
      is_free[k] = __ballot_sync(0xffffffffu, ahead[k] == 0);
      mine += __popc(is_free[k]);
    }
    load_counts(p.ref_counts, b0 + kScanStep + first, p.num_blocks, ahead);
    int total;
    int rank = found + cta_scan(lane == 0 ? mine : 0, s_warp, total);
    rank = __shfl_sync(0xffffffffu, rank, 0);
#pragma unroll
    for (int k = 0; k < kScanRows; ++k) {
      const int at = rank + __popc(is_free[k] & ((1u << lane) - 1));
      if (((is_free[k] >> lane) & 1u) && at < want) ws.free_ids[at] = static_cast<int>(b0 + first) + 32 * k;
      rank += __popc(is_free[k]);
    }
    found += total;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kPlanThreads) {
    int4 e = ws.entry[i];
    int id = -1;
    if (e.z >= 0) {
      if (e.w >= 0) {
        if (e.w < found) {
          id = ws.free_ids[e.w];
        } else {
          e.z = -1;
          report(AEG_DEVERR_POOL_EMPTY);
        }
      }
      e.w = id;
      ws.entry[i] = e;
      p.seq_lens[e.y] = max(e.z, 0);
    }
    new_blocks[i] = id;
  }
}

template <bool kVec>
__global__ void __launch_bounds__(kCopyThreads) fork_apply_kernel(const PoolParams p, int n, ForkScratch ws) {
  pdl_enter();
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int4 e = ws.entry[i];
    const int* from = p.tables + static_cast<int64_t>(e.x) * p.table_stride;
    int* to = p.tables + static_cast<int64_t>(e.y) * p.table_stride;
    const int nb = (max(e.z, 0) + kBlockTokens - 1) / kBlockTokens;
    for (int j = threadIdx.x; j < nb; j += kCopyThreads) {
      const int id = (j == nb - 1 && e.w >= 0) ? e.w : from[j];
      to[j] = id;
      if (!valid_id(id, p.num_blocks)) report(AEG_DEVERR_BLOCK_ID_RANGE);
      else if (atomicAdd(&p.ref_counts[id], 1) <= 0 && id != e.w) report(AEG_DEVERR_POOL_ENTRY);  // a free block in a row
    }
  }
  const int64_t items = n * p.segs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t i = item / p.segs;
    const int4 e = ws.entry[i];
    if (e.z < 0 || e.w < 0) continue;
    copy_segment<kVec>(p.pool + ws.tail[i] * p.block_bytes, p.pool + e.w * p.block_bytes, p.block_bytes, item - i * p.segs);
  }
}

// ---- free --------------------------------------------------------------------------------------

// One CTA a row. The row's length is taken with an exchange, so a row named twice is freed once.
__global__ void __launch_bounds__(kCopyThreads)
free_kernel(const PoolParams p, const int64_t* row_ids) {
  __shared__ int s_len;
  pdl_enter();
  const int64_t row = row_ids[blockIdx.x];
  if (!valid_id(row, p.rows)) {
    if (threadIdx.x == 0) report(AEG_DEVERR_POOL_ENTRY);
    return;
  }
  const int cap = p.table_stride * kBlockTokens;
  if (threadIdx.x == 0) {
    int len = atomicExch(&p.seq_lens[row], 0);
    if (len < 0 || len > cap) {
      report(AEG_DEVERR_SEQ_LEN_RANGE);
      len = len < 0 ? 0 : cap;
    }
    s_len = len;
  }
  __syncthreads();
  const int nb = (s_len + kBlockTokens - 1) / kBlockTokens;
  const int* ids = p.tables + row * p.table_stride;
  for (int j = threadIdx.x; j < nb; j += kCopyThreads) {
    const int id = ids[j];
    if (!valid_id(id, p.num_blocks)) {
      report(AEG_DEVERR_BLOCK_ID_RANGE);
    } else if (atomicSub(&p.ref_counts[id], 1) <= 0) {
      atomicAdd(&p.ref_counts[id], 1);  // no reference was left to give back
      report(AEG_DEVERR_POOL_ENTRY);
    }
  }
}

// ---- compact -----------------------------------------------------------------------------------

struct CompactScratch {
  int* moves;  // [0] number of moves
  int* list;   // the free ids below the number of live blocks, then the live ids from it on
};

struct CompactOut {
  int* tables;
  int* ref_counts;
  int* remap;
  int* num_live;
};

__global__ void __launch_bounds__(kPlanThreads, 1)
compact_plan_kernel(const PoolParams p, CompactScratch ws, CompactOut out) {
  __shared__ int s_warp[32];
  pdl_enter();
  const int tid = threadIdx.x;
  const int lane = tid & 31;
  const int64_t first = int64_t(tid >> 5) * 32 * kScanRows + lane;
  int rc[kScanRows], ahead[kScanRows];
  int mine = 0, n_live = 0;
  for (int64_t b0 = 0; b0 < p.num_blocks; b0 += kScanStep) {
    load_counts(p.ref_counts, b0 + first, p.num_blocks, rc);
#pragma unroll
    for (int k = 0; k < kScanRows; ++k) mine += rc[k] > 0;
  }
  load_counts(p.ref_counts, first, p.num_blocks, ahead);
  cta_scan(mine, s_warp, n_live);
  // There are as many free ids below n_live as live ones from it on: listed in order of id, the
  // former fill the list's first half, the latter its second.
  int listed = 0;
  for (int64_t b0 = 0; b0 < p.num_blocks; b0 += kScanStep) {
    const int64_t b = b0 + first;
    uint32_t in_list[kScanRows];
    int count = 0;
#pragma unroll
    for (int k = 0; k < kScanRows; ++k) {
      rc[k] = ahead[k];
      const int64_t id = b + 32 * k;
      in_list[k] = __ballot_sync(0xffffffffu, id < p.num_blocks && (id < n_live) == (rc[k] <= 0));
      count += __popc(in_list[k]);
    }
    load_counts(p.ref_counts, b + kScanStep, p.num_blocks, ahead);
    int total;
    int at = listed + cta_scan(lane == 0 ? count : 0, s_warp, total);
    at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
    for (int k = 0; k < kScanRows; ++k) {
      const int id = static_cast<int>(b) + 32 * k;
      if (b + 32 * k < p.num_blocks) {
        const bool low = id < n_live, live = rc[k] > 0;
        const int place = at + __popc(in_list[k] & ((1u << lane) - 1));
        if (low != live) ws.list[place] = id;
        // A moving block's place in the list until compact_apply_kernel puts its new id there.
        out.remap[id] = !live ? -1 : (low ? id : -2 - place);
        out.ref_counts[id] = low ? max(rc[k], 0) : 0;
      }
      at += __popc(in_list[k]);
    }
    listed += total;
  }
  const int moves = listed / 2;
  if (tid == 0) {
    ws.moves[0] = moves;
    out.num_live[0] = n_live;
  }
}

template <bool kVec>
__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(const PoolParams p, CompactScratch ws, CompactOut out) {
  pdl_enter();
  const int cap = p.table_stride * kBlockTokens;
  const int moves = ws.moves[0];
  // Rows read remap while moving blocks' entries go from a place in the list to the id it stands for: either
  // says the same, and relaxed accesses see one of them whole.
  for (int r = blockIdx.x * kCopyThreads + threadIdx.x; r < moves; r += gridDim.x * kCopyThreads) {
    const int to = ws.list[r], from = ws.list[moves + r];
    st_relaxed(&out.remap[from], to);
    out.ref_counts[to] = p.ref_counts[from];
  }
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
    int len = p.seq_lens[row];
    if (len < 0 || len > cap) {
      if (threadIdx.x == 0) report(AEG_DEVERR_SEQ_LEN_RANGE);
      len = len < 0 ? 0 : cap;
    }
    const int nb = (len + kBlockTokens - 1) / kBlockTokens;
    const int64_t base = static_cast<int64_t>(row) * p.table_stride;
    for (int j = threadIdx.x; j < p.table_stride; j += kCopyThreads) {
      int id = p.tables[base + j];
      if (j < nb) {
        int to = valid_id(id, p.num_blocks) ? ld_relaxed(&out.remap[id]) : -1;
        if (to < -1) to = ws.list[-2 - to - moves];
        if (to >= 0) id = to;
        else report(AEG_DEVERR_BLOCK_ID_RANGE);
      }
      out.tables[base + j] = id;
    }
  }
  const int64_t items = moves * p.segs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r = item / p.segs;
    copy_segment<kVec>(p.pool + ws.list[moves + r] * p.block_bytes, p.pool + ws.list[r] * p.block_bytes, p.block_bytes,
                       item - r * p.segs);
  }
}

// ---- host --------------------------------------------------------------------------------------

inline size_t align16(size_t x) { return (x + 15) & ~size_t(15); }

size_t fork_scratch(void* base, int64_t n, ForkScratch* ws) {
  char* b = static_cast<char*>(base);
  size_t off = 0;
  if (ws) ws->entry = reinterpret_cast<int4*>(b + off);
  off += sizeof(int4) * n;
  if (ws) ws->tail = reinterpret_cast<int*>(b + off);
  off = align16(off + sizeof(int) * n);
  if (ws) ws->free_ids = reinterpret_cast<int*>(b + off);
  return align16(off + sizeof(int) * n);
}

int check_pool(const char* what, PoolParams& p, void* pool, size_t block_bytes, int64_t num_blocks, int32_t* ref_counts,
               int32_t* tables, int table_stride, int rows, int32_t* seq_lens) {
  AEG_CHECK_ARG(num_blocks >= 0 && num_blocks <= (1LL << 30), "%s: num_blocks %lld out of range", what, (long long)num_blocks);
  AEG_CHECK_ARG(rows >= 0 && table_stride > 0 && table_stride <= (1 << 26), "%s: bad table shape [%d, %d]", what, rows,
                table_stride);
  AEG_CHECK_ARG(num_blocks == 0 || ref_counts != nullptr, "%s: ref_counts is NULL", what);
  AEG_CHECK_ARG(rows == 0 || (tables != nullptr && seq_lens != nullptr), "%s: null table or length pointer", what);
  AEG_CHECK_ARG(aligned(ref_counts, 4) && aligned(tables, 4) && aligned(seq_lens, 4), "%s: int32 arrays must be aligned", what);
  p.pool = static_cast<uint8_t*>(pool);
  p.block_bytes = static_cast<int64_t>(block_bytes);
  p.segs = (p.block_bytes + kSegVecs * 16 - 1) / (kSegVecs * 16);
  p.num_blocks = static_cast<int>(num_blocks);
  p.ref_counts = ref_counts;
  p.tables = tables;
  p.table_stride = table_stride;
  p.rows = rows;
  p.seq_lens = seq_lens;
  return AEG_OK;
}

template <typename... Params, typename... Args>
cudaError_t launch(void (*kern)(Params...), int64_t grid, int threads, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

bool vectors(const PoolParams& p) { return p.block_bytes % 16 == 0 && aligned(p.pool, 16); }

}  // namespace

uint32_t deverr_read_and_clear_pool(cudaStream_t s, cudaError_t* err) {
  uint32_t v = 0, zero = 0;
  *err = cudaMemcpyFromSymbolAsync(&v, g_deverr_pool, sizeof(v), 0, cudaMemcpyDeviceToHost, s);
  if (*err == cudaSuccess) *err = cudaStreamSynchronize(s);
  if (*err == cudaSuccess) *err = cudaMemcpyToSymbolAsync(g_deverr_pool, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
  if (*err == cudaSuccess) *err = cudaStreamSynchronize(s);
  return v;
}

}  // namespace aeg

extern "C" {

size_t aeg_fork_blocks_workspace_size(int64_t n) { return n <= 0 ? 0 : aeg::fork_scratch(nullptr, n, nullptr); }

int aeg_fork_blocks(void* pool, size_t block_bytes, int64_t num_blocks, int32_t* ref_counts, int32_t* block_tables,
                    int table_stride, int rows, int32_t* seq_lens, const int64_t* d_src_rows, const int64_t* d_dst_rows,
                    int64_t n, int32_t* new_blocks, void* workspace, size_t workspace_bytes, void* stream) {
  aeg::PoolParams p{};
  const int st = aeg::check_pool("fork_blocks", p, pool, block_bytes, num_blocks, ref_counts, block_tables, table_stride,
                                 rows, seq_lens);
  if (st != AEG_OK) return st;
  AEG_CHECK_ARG(n >= 0 && n <= (1LL << 24), "fork_blocks: entry count %lld out of range", (long long)n);
  if (n == 0) return AEG_OK;
  AEG_CHECK_ARG(d_src_rows && d_dst_rows && new_blocks && (pool || num_blocks == 0), "fork_blocks: null pointer");
  AEG_CHECK_ARG(aeg::aligned(d_src_rows, 8) && aeg::aligned(d_dst_rows, 8) && aeg::aligned(new_blocks, 4),
                "fork_blocks: misaligned id array");
  AEG_CHECK_ARG(workspace != nullptr && aeg::aligned(workspace, 16) && workspace_bytes >= aeg_fork_blocks_workspace_size(n),
                "fork_blocks: workspace of %zu bytes, need %zu, 16-byte aligned", workspace_bytes,
                aeg_fork_blocks_workspace_size(n));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  aeg::ForkScratch ws{};
  aeg::fork_scratch(workspace, n, &ws);
  AEG_CHECK_CUDA(aeg::launch(aeg::fork_plan_kernel, 1, aeg::kPlanThreads, s, p, d_src_rows, d_dst_rows,
                             static_cast<int>(n), ws, new_blocks));
  const int64_t grid = std::min<int64_t>(n * std::max<int64_t>(p.segs, 1), int64_t(aeg::num_sms()) * 8);
  AEG_CHECK_CUDA(aeg::launch(aeg::vectors(p) ? aeg::fork_apply_kernel<true> : aeg::fork_apply_kernel<false>, grid,
                             aeg::kCopyThreads, s, p, static_cast<int>(n), ws));
  AEG_CHECK_LAUNCH("fork_blocks");
  aeg::note_launch(s, false);
  return AEG_OK;
}

int aeg_free_blocks(int64_t num_blocks, int32_t* ref_counts, const int32_t* block_tables, int table_stride, int rows,
                    int32_t* seq_lens, const int64_t* d_rows, int64_t n, void* stream) {
  aeg::PoolParams p{};
  const int st = aeg::check_pool("free_blocks", p, nullptr, 0, num_blocks, ref_counts, const_cast<int32_t*>(block_tables),
                                 table_stride, rows, seq_lens);
  if (st != AEG_OK) return st;
  AEG_CHECK_ARG(n >= 0 && n <= (1LL << 24), "free_blocks: row count %lld out of range", (long long)n);
  if (n == 0) return AEG_OK;
  AEG_CHECK_ARG(d_rows != nullptr && aeg::aligned(d_rows, 8), "free_blocks: null or misaligned row array");
  AEG_CHECK_CUDA(aeg::launch(aeg::free_kernel, n, aeg::kCopyThreads, static_cast<cudaStream_t>(stream), p, d_rows));
  AEG_CHECK_LAUNCH("free_blocks");
  aeg::note_launch(static_cast<cudaStream_t>(stream), false);
  return AEG_OK;
}

size_t aeg_compact_blocks_workspace_size(int64_t num_blocks) {
  return num_blocks < 0 ? 0 : 16 + aeg::align16(sizeof(int32_t) * size_t(num_blocks));
}

int aeg_compact_blocks(void* pool, size_t block_bytes, int64_t num_blocks, const int32_t* ref_counts,
                       const int32_t* block_tables, int table_stride, int rows, const int32_t* seq_lens,
                       int32_t* ref_counts_out, int32_t* block_tables_out, int32_t* remap, int32_t* num_live,
                       void* workspace, size_t workspace_bytes, void* stream) {
  aeg::PoolParams p{};
  const int st = aeg::check_pool("compact_blocks", p, pool, block_bytes, num_blocks, const_cast<int32_t*>(ref_counts),
                                 const_cast<int32_t*>(block_tables), table_stride, rows, const_cast<int32_t*>(seq_lens));
  if (st != AEG_OK) return st;
  AEG_CHECK_ARG(num_live != nullptr && (num_blocks == 0 || (pool && ref_counts_out && remap)) &&
                    (rows == 0 || block_tables_out),
                "compact_blocks: null pointer");
  AEG_CHECK_ARG(ref_counts_out != ref_counts || num_blocks == 0, "compact_blocks: ref_counts_out must not be ref_counts");
  AEG_CHECK_ARG(aeg::aligned(ref_counts_out, 4) && aeg::aligned(block_tables_out, 4) && aeg::aligned(remap, 4) &&
                    aeg::aligned(num_live, 4),
                "compact_blocks: int32 arrays must be aligned");
  AEG_CHECK_ARG(workspace != nullptr && aeg::aligned(workspace, 16) &&
                    workspace_bytes >= aeg_compact_blocks_workspace_size(num_blocks),
                "compact_blocks: workspace of %zu bytes, need %zu, 16-byte aligned", workspace_bytes,
                aeg_compact_blocks_workspace_size(num_blocks));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  aeg::CompactScratch ws{static_cast<int*>(workspace), reinterpret_cast<int*>(static_cast<char*>(workspace) + 16)};
  aeg::CompactOut out{block_tables_out, ref_counts_out, remap, num_live};
  AEG_CHECK_CUDA(aeg::launch(aeg::compact_plan_kernel, 1, aeg::kPlanThreads, s, p, ws, out));
  // At most half of the blocks move: free ones below the number of live ones, one for each live one beyond.
  const int64_t work = std::max<int64_t>(num_blocks / 2 * std::max<int64_t>(p.segs, 1), rows);
  const int64_t grid = std::max<int64_t>(std::min<int64_t>(work, int64_t(aeg::num_sms()) * 8), 1);
  AEG_CHECK_CUDA(aeg::launch(aeg::vectors(p) ? aeg::compact_apply_kernel<true> : aeg::compact_apply_kernel<false>, grid,
                             aeg::kCopyThreads, s, p, ws, out));
  AEG_CHECK_LAUNCH("compact_blocks");
  aeg::note_launch(s, false);
  return AEG_OK;
}

}  // extern "C"
