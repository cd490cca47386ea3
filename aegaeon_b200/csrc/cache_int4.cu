// The 4-bit KV cache's write (reshape_and_cache_int4) and read-back (gather_cache_int4).
//
// The write is reshape_and_cache (cache_write.cu) with the rows rounded to 4 bits: slot s is row
// s % 16 of the tiles of block s / 16, a slot < 0 is padding. Format and layout: int4_tile.cuh.
// Both are bound by memory: 512 bytes of keys and values a (token, head) on one side, 144 bytes of
// codes and pairs on the other. One warp moves one (token, head): lanes 0..15 its key, 16..31 its
// value, 8 dims a lane (one 16-byte vector), 8 lanes a 64-dim group, so that a group's range is
// three shuffles away and a lane's codes are exactly one key word or two value halves. Where there are
// enough of them a warp takes kTokens tokens x kHeads heads at a time, all loads before the first use; the
// heads' chunks are the grid's second dimension, so that no index is divided.
//
// Measured (device time in a graph of calls over more data than L2 holds): a prompt batch of 11,348 tokens x
// 4 heads is written in 13.0 us in bf16 (2.3 TB/s; 11.0 us with the scale and codes made up, so the rounding
// costs little), 14.7 us in fp16, of whose warps 21 % take the general form on N(0, 1) rows (bf16 3 %), and
// read back in 9.5 us (3.2 TB/s), 2.1 to 3.2 times what the bytes need: every lane stores or loads 4 to 8 bytes of
// a tile where it is, although a prompt fills whole tiles, which could go through shared memory. 64 tokens
// take 1.8 us and 1024 slots 2.4 us, a launch each.
#include "int4_tile.cuh"

#include <algorithm>

namespace aeg {
namespace {

__device__ unsigned int g_deverr_int4 = 0;

constexpr int kThreads = 128;
constexpr int kWarpsPerCta = kThreads / 32;

// A lane's 8 elements of a row: one 16-byte vector, or 8 loads where rows are not 16-byte aligned.
template <bool kVec>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
  if constexpr (kVec) {
    return *reinterpret_cast<const uint4*>(p);
  } else {
    return make_uint4(p[0] | (uint32_t(p[1]) << 16), p[2] | (uint32_t(p[3]) << 16), p[4] | (uint32_t(p[5]) << 16),
                      p[6] | (uint32_t(p[7]) << 16));
  }
}

template <bool kVec>
__device__ __forceinline__ void store8(uint16_t* p, const uint4& v) {
  if constexpr (kVec) {
    *reinterpret_cast<uint4*>(p) = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[2 * i] = static_cast<uint16_t>(w[i]);
      p[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
    }
  }
}

struct Rows {
  uint16_t* key;
  uint16_t* value;
  int64_t key_stride;    // elements between tokens
  int64_t value_stride;
  uint8_t* cache;        // the layer's first tile
  int64_t block_stride;  // bytes between blocks
  const int64_t* slots;
  int64_t num_slots;
  int64_t tokens;
  int heads;
  bool early;  // of a write: let the next kernel launch before the wait
};

template <typename T, bool kVec, int kTokens, int kHeads>
__global__ void __launch_bounds__(kThreads) write_int4_kernel(const Rows p) {
  constexpr int kItems = kTokens * kHeads;
  pdl_enter_write(p.early);
  const int lane = threadIdx.x & 31, l = lane & 15;
  const bool is_key = lane < 16;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarpsPerCta * kTokens;
  const int h0 = blockIdx.y * kHeads;
  const int64_t stride = is_key ? p.key_stride : p.value_stride;
  const uint16_t* rows = (is_key ? p.key : p.value) + h0 * kInt4Dim + 8 * l;
  uint8_t* tiles = p.cache + static_cast<int64_t>(h0) * kInt4TileBytes;
  const int pairs_at = (is_key ? kInt4KeyPairs : kInt4ValuePairs) + (l >> 3) * 4;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5)) * kTokens; t0 < p.tokens; t0 += step) {
    uint4 v[kItems];
    int64_t slot[kTokens];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int64_t t = t0 + k / kHeads;
      const bool there = t < p.tokens && h0 + k % kHeads < p.heads;
      if (k % kHeads == 0) slot[k / kHeads] = t < p.tokens ? p.slots[t] : -1;
      v[k] = there ? load8<kVec>(rows + t * stride + (k % kHeads) * kInt4Dim) : make_uint4(0u, 0u, 0u, 0u);
    }
    // Tokens of one word pair (an even slot and the next one) are stored together: 4-byte words of both
    // instead of 2-byte halves of each.
    bool pair = kTokens % 2 == 0;
#pragma unroll
    for (int j = 0; j < kTokens; ++j) {
      if (slot[j] >= p.num_slots) {
        if (lane == 0) atomicOr(&g_deverr_int4, AEG_DEVERR_SLOT_RANGE);
        slot[j] = -1;
      }
      if (j % 2) pair = pair && slot[j - 1] >= 0 && !(slot[j - 1] & 1) && slot[j] == slot[j - 1] + 1;
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (h0 + i >= p.heads) break;
      uint2 q[kTokens];
#pragma unroll
      for (int j = 0; j < kTokens; ++j) q[j] = int4_quantise<T>(v[j * kHeads + i]);
#pragma unroll
      for (int j = 0; j < kTokens; ++j) {
        if (slot[j] < 0) continue;
        const int t = static_cast<int>(slot[j] & 15);
        uint8_t* tile = tiles + (slot[j] >> 4) * p.block_stride + i * kInt4TileBytes;
        if ((l & 7) == 0) *reinterpret_cast<uint32_t*>(tile + pairs_at + t * 8) = q[j].y;
        if (!pair) {
          // A key lane's word as two halves beside each other, a value lane's 4 bytes apart.
          uint16_t* half = reinterpret_cast<uint16_t*>(tile + (is_key ? int4_key_word(t, l) : int4_value_half(t, l)));
          half[0] = static_cast<uint16_t>(q[j].x);
          half[is_key ? 1 : 2] = static_cast<uint16_t>(q[j].x >> 16);
        } else if (j % 2 == 0) {
          const uint32_t a = q[j].x, b = q[(j + 1) % kTokens].x;
          uint32_t* word = reinterpret_cast<uint32_t*>(tile + (is_key ? int4_key_word(t, l) : int4_value_half(t, l)));
          word[0] = is_key ? a : __byte_perm(a, b, 0x5410);
          word[is_key ? 16 : 1] = is_key ? b : __byte_perm(a, b, 0x7632);  // the next token's key row is 64 bytes on
        }
      }
    }
  }
}

template <typename T, bool kVec, int kTokens, int kHeads>
__global__ void __launch_bounds__(kThreads) gather_int4_kernel(const Rows p) {
  constexpr int kItems = kTokens * kHeads;
  pdl_enter();
  const int lane = threadIdx.x & 31, l = lane & 15;
  const bool is_key = lane < 16;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarpsPerCta * kTokens;
  const int h0 = blockIdx.y * kHeads;
  const int64_t stride = is_key ? p.key_stride : p.value_stride;
  uint16_t* rows = (is_key ? p.key : p.value) + h0 * kInt4Dim + 8 * l;
  const uint8_t* tiles = p.cache + static_cast<int64_t>(h0) * kInt4TileBytes;
  const int pairs_at = (is_key ? kInt4KeyPairs : kInt4ValuePairs) + (l >> 3) * 4;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5)) * kTokens; t0 < p.tokens; t0 += step) {
    uint32_t word[kItems], pair[kItems];
    int64_t slot[kTokens];
#pragma unroll
    for (int j = 0; j < kTokens; ++j) {
      slot[j] = t0 + j < p.tokens ? p.slots[t0 + j] : -1;
      if (slot[j] >= p.num_slots && lane == 0) atomicOr(&g_deverr_int4, AEG_DEVERR_SLOT_RANGE);
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      word[k] = 0;
      pair[k] = 0;  // scale 0, minimum 0: zeros
      const int64_t s = slot[k / kHeads];
      if (s >= 0 && s < p.num_slots && h0 + k % kHeads < p.heads) {
        const int t = static_cast<int>(s & 15);
        const uint8_t* tile = tiles + (s >> 4) * p.block_stride + (k % kHeads) * kInt4TileBytes;
        // The 8 bytes around a key lane's word, or a value lane's two words with both tokens' halves.
        const int at = is_key ? int4_key_word(t, l) : int4_value_half(t, l);
        const uint2 two = *reinterpret_cast<const uint2*>(tile + (at & ~7));
        word[k] = is_key ? (at & 4 ? two.y : two.x) : __byte_perm(two.x, two.y, t & 1 ? 0x7632 : 0x5410);
        pair[k] = *reinterpret_cast<const uint32_t*>(tile + pairs_at + t * 8);
      }
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int64_t t = t0 + k / kHeads;
      if (t >= p.tokens || h0 + k % kHeads >= p.heads) continue;
      const float2 sm = unpack2<T>(pair[k]);
      // One rounding to fp32 (code * scale alone is exact), one to the type.
      auto value = [&](int n) { return fmaf(static_cast<float>((word[k] >> (4 * n)) & 15u), sm.x, sm.y); };
      store8<kVec>(rows + t * stride + (k % kHeads) * kInt4Dim,
                   make_uint4(pack2<T>(value(0), value(1)), pack2<T>(value(2), value(3)), pack2<T>(value(4), value(5)),
                              pack2<T>(value(6), value(7))));
    }
  }
}

// Checks shared by both directions; fills `p`.
int prepare(const char* what, Rows& p, const void* key, const void* value, int64_t key_stride, int64_t value_stride,
            const void* cache, int64_t block_stride, int64_t num_blocks, const int64_t* slot_mapping, int64_t T, int Hkv,
            int D, int dtype) {
  AEG_CHECK_ARG(T >= 0 && T <= 0x7fffffffLL, "%s: token count %lld out of range", what, (long long)T);
  AEG_CHECK_ARG(Hkv > 0 && D > 0, "%s: Hkv and D must be positive", what);
  if (D != kInt4Dim) return set_error(AEG_ERR_UNSUPPORTED, "%s: head_dim %d not supported (only 128)", what, D);
  AEG_CHECK_ARG(dtype == AEG_DTYPE_FP16 || dtype == AEG_DTYPE_BF16, "%s: dtype %d is not fp16/bf16", what, dtype);
  AEG_CHECK_ARG(num_blocks >= 0 && num_blocks <= 0x7fffffffLL, "%s: num_blocks %lld out of range", what, (long long)num_blocks);
  if (T == 0) return AEG_OK;
  AEG_CHECK_ARG(key && value && cache && slot_mapping, "%s: null pointer", what);
  const int64_t row = int64_t(Hkv) * D;
  AEG_CHECK_ARG(key_stride >= row && value_stride >= row, "%s: token stride smaller than Hkv*D", what);
  AEG_CHECK_ARG(block_stride >= int64_t(Hkv) * kInt4TileElems && block_stride % 8 == 0,
                "%s: block stride must be a multiple of 8 elements and >= Hkv*1152", what);
  AEG_CHECK_ARG(aligned(cache, 16), "%s: the cache must be 16-byte aligned", what);
  AEG_CHECK_ARG(aligned(key, 2) && aligned(value, 2) && aligned(slot_mapping, 8), "%s: misaligned pointer", what);
  p.key = static_cast<uint16_t*>(const_cast<void*>(key));
  p.value = static_cast<uint16_t*>(const_cast<void*>(value));
  p.key_stride = key_stride;
  p.value_stride = value_stride;
  p.cache = static_cast<uint8_t*>(const_cast<void*>(cache));
  p.block_stride = 2 * block_stride;
  p.slots = slot_mapping;
  p.num_slots = num_blocks * 16;
  p.tokens = T;
  p.heads = Hkv;
  return AEG_OK;
}

using Kernel = void (*)(const Rows);

template <typename T, int kTokens, int kHeads>
Kernel pick(bool write, bool vec) {
  if (write) return vec ? write_int4_kernel<T, true, kTokens, kHeads> : write_int4_kernel<T, false, kTokens, kHeads>;
  return vec ? gather_int4_kernel<T, true, kTokens, kHeads> : gather_int4_kernel<T, false, kTokens, kHeads>;
}

// Several (token, head) a warp only where every resident warp has as many; then 4, of two tokens (which
// often share their words) where there are 2 heads.
template <typename T>
Kernel pick(bool write, bool vec, int64_t items, int heads, int* tokens, int* chunk) {
  const bool many = items >= int64_t(num_sms()) * 16 * kWarpsPerCta;
  *chunk = !many || heads == 1 ? 1 : 2;
  *tokens = many ? 4 / *chunk : 1;
  if (!many) return pick<T, 1, 1>(write, vec);
  return heads == 1 ? pick<T, 4, 1>(write, vec) : pick<T, 2, 2>(write, vec);
}

int launch(const char* what, bool write, Rows& p, int dtype, cudaStream_t stream) {
  const bool vec = aligned(p.key, 16) && aligned(p.value, 16) && p.key_stride % 8 == 0 && p.value_stride % 8 == 0;
  int tokens = 1, chunk = 1;
  const Kernel k = dtype == AEG_DTYPE_BF16 ? pick<__nv_bfloat16>(write, vec, p.tokens * p.heads, p.heads, &tokens, &chunk)
                                           : pick<__half>(write, vec, p.tokens * p.heads, p.heads, &tokens, &chunk);
  const int chunks = (p.heads + chunk - 1) / chunk;
  AEG_CHECK_ARG(chunks <= 65535, "%s: %d KV heads are too many", what, p.heads);
  const int64_t per_cta = int64_t(kWarpsPerCta) * tokens;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  const int64_t most = std::max<int64_t>(int64_t(num_sms()) * 256 / chunks, 1);
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>((p.tokens + per_cta - 1) / per_cta, most)),
                     static_cast<unsigned>(chunks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  p.early = write && follows_attention(stream);
  AEG_CHECK_CUDA(cudaLaunchKernelEx(&cfg, k, p));
  AEG_CHECK_LAUNCH(what);
  note_launch(stream, false);
  return AEG_OK;
}

}  // namespace

uint32_t deverr_read_and_clear_int4(cudaStream_t s, cudaError_t* err) {
  uint32_t v = 0, zero = 0;
  *err = cudaMemcpyFromSymbolAsync(&v, g_deverr_int4, sizeof(v), 0, cudaMemcpyDeviceToHost, s);
  if (*err == cudaSuccess) *err = cudaStreamSynchronize(s);
  if (*err == cudaSuccess) *err = cudaMemcpyToSymbolAsync(g_deverr_int4, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
  if (*err == cudaSuccess) *err = cudaStreamSynchronize(s);
  return v;
}

}  // namespace aeg

extern "C" {

int aeg_reshape_and_cache_int4(const void* key, const void* value, int64_t key_stride, int64_t value_stride,
                               void* kv_cache, int64_t block_stride, int64_t num_blocks, const int64_t* slot_mapping,
                               int64_t T, int Hkv, int D, int dtype, void* stream) {
  aeg::Rows p{};
  const int st = aeg::prepare("reshape_and_cache_int4", p, key, value, key_stride, value_stride, kv_cache, block_stride,
                              num_blocks, slot_mapping, T, Hkv, D, dtype);
  if (st != AEG_OK || T == 0) return st;
  return aeg::launch("reshape_and_cache_int4", true, p, dtype, static_cast<cudaStream_t>(stream));
}

int aeg_gather_cache_int4(void* key, void* value, int64_t key_stride, int64_t value_stride, const void* kv_cache,
                          int64_t block_stride, int64_t num_blocks, const int64_t* slot_mapping, int64_t T, int Hkv,
                          int D, int dtype, void* stream) {
  aeg::Rows p{};
  const int st = aeg::prepare("gather_cache_int4", p, key, value, key_stride, value_stride, kv_cache, block_stride,
                              num_blocks, slot_mapping, T, Hkv, D, dtype);
  if (st != AEG_OK || T == 0) return st;
  return aeg::launch("gather_cache_int4", false, p, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
