// Rotary positions with several axes (time, height, width), applied to queries and keys.
//
// For frequency i < half of a token with positions pos[a], a = axis(i):
//   theta = pos[a] * inv_freq[i]
//   out[i]        = x[i] cos(theta) - x[i + half] sin(theta)
//   out[i + half] = x[i + half] cos(theta) + x[i] sin(theta)
// and dims from 2 * half on are copied. A text model's single axis is the case of one section.
//
// The rows are read once and written once, so memory bounds it. What has to stay small beside that
// is the angles: they are the same for every head of a token, so one CTA takes a whole token, its
// first `half` threads compute one cosine and sine each into shared memory while the rows' loads
// are in flight, and all threads then rotate the token's heads. An fp32 angle would be off by
// 2^-24 * theta (6e-3 at position 100,000), so the turn theta / 2 pi is made and reduced to
// [-1/2, 1/2] in 64 bits (error below 1e-10 turns at 2^20) and only the reduced turn goes to the
// fp32 sine and cosine. The next token's first vectors and position are loaded before this token's barrier:
// 11,348 tokens of 28 + 4 heads run 32.8 us (5.7 TB/s, 0.87 of the measured copy rate; 39.3 us without),
// a decode batch of 256 tokens x 36 heads 3.9 us.
#include "aeg_common.cuh"

#include <algorithm>

namespace aeg {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;
constexpr int kAxisWords = kMaxHalf / 16;  // 2 bits a frequency

struct RotaryParams {
  const uint16_t* x[2];  // queries, keys
  uint16_t* out[2];
  int64_t x_stride[2];  // elements between tokens
  int64_t out_stride[2];
  int heads[2];
  const int64_t* positions;  // [axes, tokens]
  int64_t axis_stride;
  const float* inv_freq;
  float scaling;
  int half;
  int dim;
  int64_t tokens;
  uint32_t axis[kAxisWords];
};

template <int kVec>
struct Vec;
template <>
struct Vec<8> {
  using Type = uint4;
};
template <>
struct Vec<1> {
  using Type = uint16_t;
};

template <typename T, int kVec>
__device__ __forceinline__ void to_floats(const typename Vec<kVec>::Type& v, float (&f)[kVec]) {
  if constexpr (kVec == 8) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = unpack2<T>(w[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  } else {
    f[0] = unpack2<T>(v).x;
  }
}

template <typename T, int kVec>
__device__ __forceinline__ typename Vec<kVec>::Type from_floats(const float (&f)[kVec]) {
  if constexpr (kVec == 8) {
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  } else {
    return static_cast<uint16_t>(pack2<T>(f[0], 0.f));
  }
}

template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  using V = typename Vec<kVec>::Type;
  __shared__ float s_cos[2][kMaxHalf], s_sin[2][kMaxHalf];
  pdl_enter();
  const int tid = threadIdx.x;
  const int per_head = p.half / kVec;            // rotated vectors of a head (each with its partner)
  const int rest = p.dim / kVec - 2 * per_head;  // copied vectors of a head
  const int n_rot = (p.heads[0] + p.heads[1]) * per_head;
  const int n_rest = (p.heads[0] + p.heads[1]) * rest;
  double turn_per_pos = 0.0;
  const int64_t* pos = p.positions;
  if (tid < p.half) {
    turn_per_pos = static_cast<double>(p.inv_freq[tid]) * 0.15915494309189535;  // 1 / (2 pi)
    pos += static_cast<int64_t>((p.axis[tid >> 4] >> (2 * (tid & 15))) & 3u) * p.axis_stride;
  }
  // A thread's vectors: item k is head k / per_head, vector k % per_head of it, `off` elements into the
  // token's row of queries or keys.
  auto locate = [&](int k, int per, int base, int& which, int& c) {
    const int head = k / per;
    c = k - head * per;
    which = head >= p.heads[0] ? 1 : 0;
    return (which ? head - p.heads[0] : head) * p.dim + base + c * kVec;
  };
  auto source = [&](int which, int64_t t, int off) {
    return reinterpret_cast<const V*>((which ? p.x[1] : p.x[0]) + t * (which ? p.x_stride[1] : p.x_stride[0]) + off);
  };
  auto target = [&](int which, int64_t t, int off) {
    return reinterpret_cast<V*>((which ? p.out[1] : p.out[0]) + t * (which ? p.out_stride[1] : p.out_stride[0]) + off);
  };
  // The first item of the next token and its position are loaded while this one is rotated.
  int which0 = 0, c0 = 0;
  const int off0 = tid < n_rot ? locate(tid, per_head, 0, which0, c0) : 0;
  V a0{}, b0{};
  int64_t at = 0;
  auto load_first = [&](int64_t t) {
    if (t >= p.tokens) return;
    if (tid < n_rot) {
      const V* src = source(which0, t, off0);
      a0 = src[0];
      b0 = src[per_head];
    }
    if (tid < p.half) at = pos[t];
  };
  load_first(blockIdx.x);
  int buf = 0;
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x, buf ^= 1) {
    if (tid < p.half) {
      const double turn = turn_per_pos * static_cast<double>(at);
      float sn, cs;
      sincospif(2.f * static_cast<float>(turn - rint(turn)), &sn, &cs);
      s_cos[buf][tid] = cs * p.scaling;
      s_sin[buf][tid] = sn * p.scaling;
    }
    V a = a0, b = b0;
    load_first(t + gridDim.x);
    // One barrier a token: the buffers alternate, and a thread passes the next token's barrier only
    // when all threads have left this token's rotations behind.
    __syncthreads();
    int which = which0, c = c0, off = off0;
    for (int k = tid; k < n_rot; k += kThreads) {
      if (k != tid) {
        off = locate(k, per_head, 0, which, c);
        const V* src = source(which, t, off);
        a = src[0];
        b = src[per_head];
      }
      float fa[kVec], fb[kVec], oa[kVec], ob[kVec];
      to_floats<T, kVec>(a, fa);
      to_floats<T, kVec>(b, fb);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float cs = s_cos[buf][c * kVec + i], sn = s_sin[buf][c * kVec + i];
        oa[i] = fa[i] * cs - fb[i] * sn;
        ob[i] = fb[i] * cs + fa[i] * sn;
      }
      V* dst = target(which, t, off);
      dst[0] = from_floats<T, kVec>(oa);
      dst[per_head] = from_floats<T, kVec>(ob);
    }
    for (int k = tid; k < n_rest; k += kThreads) {
      off = locate(k, rest, 2 * p.half, which, c);
      target(which, t, off)[0] = source(which, t, off)[0];
    }
  }
}

}  // namespace
}  // namespace aeg

extern "C" int aeg_rotary_multi_axis(void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride, const void* q,
                                     int64_t q_stride, const void* k, int64_t k_stride, const int64_t* positions,
                                     int64_t axis_stride, int axes, const float* inv_freq, const uint8_t* axis_of,
                                     int half, float scaling, int64_t T, int Hq, int Hkv, int D, int dtype, void* stream) {
  AEG_CHECK_ARG(T >= 0 && T <= 0x7fffffffLL, "rotary_multi_axis: token count %lld out of range", (long long)T);
  AEG_CHECK_ARG(Hq > 0 && Hkv >= 0 && D > 0, "rotary_multi_axis: head counts and head_dim must be positive");
  AEG_CHECK_ARG(dtype == AEG_DTYPE_FP16 || dtype == AEG_DTYPE_BF16, "rotary_multi_axis: dtype %d is not fp16/bf16", dtype);
  AEG_CHECK_ARG(axes >= 1 && axes <= 4, "rotary_multi_axis: %d axes, 1 to 4 are supported", axes);
  AEG_CHECK_ARG(half >= 1 && 2 * half <= D, "rotary_multi_axis: %d frequencies do not fit head_dim %d", half, D);
  if (half > aeg::kMaxHalf)
    return aeg::set_error(AEG_ERR_UNSUPPORTED, "rotary_multi_axis: %d frequencies, at most %d", half, aeg::kMaxHalf);
  AEG_CHECK_ARG(int64_t(Hq + int64_t(Hkv)) * D <= (1 << 28), "rotary_multi_axis: rows of %lld elements are too long",
                (long long)(int64_t(Hq + int64_t(Hkv)) * D));
  AEG_CHECK_ARG(axis_of != nullptr, "rotary_multi_axis: axis_of is NULL");
  aeg::RotaryParams p{};
  for (int i = 0; i < half; ++i) {
    AEG_CHECK_ARG(axis_of[i] < axes, "rotary_multi_axis: frequency %d names axis %d of %d", i, int(axis_of[i]), axes);
    p.axis[i >> 4] |= uint32_t(axis_of[i]) << (2 * (i & 15));
  }
  if (T == 0) return AEG_OK;
  AEG_CHECK_ARG(q && q_out && positions && inv_freq && (Hkv == 0 || (k && k_out)), "rotary_multi_axis: null pointer");
  AEG_CHECK_ARG(q_stride >= int64_t(Hq) * D && q_out_stride >= int64_t(Hq) * D && k_stride >= int64_t(Hkv) * D &&
                    k_out_stride >= int64_t(Hkv) * D,
                "rotary_multi_axis: token stride smaller than heads*D");
  AEG_CHECK_ARG(axis_stride >= 0, "rotary_multi_axis: negative axis stride");
  AEG_CHECK_ARG(aeg::aligned(q, 2) && aeg::aligned(k, 2) && aeg::aligned(q_out, 2) && aeg::aligned(k_out, 2) &&
                    aeg::aligned(positions, 8) && aeg::aligned(inv_freq, 4),
                "rotary_multi_axis: misaligned pointer");
  p.x[0] = static_cast<const uint16_t*>(q);
  p.x[1] = static_cast<const uint16_t*>(k);
  p.out[0] = static_cast<uint16_t*>(q_out);
  p.out[1] = static_cast<uint16_t*>(k_out);
  p.x_stride[0] = q_stride;
  p.x_stride[1] = k_stride;
  p.out_stride[0] = q_out_stride;
  p.out_stride[1] = k_out_stride;
  p.heads[0] = Hq;
  p.heads[1] = Hkv;
  p.positions = positions;
  p.axis_stride = axis_stride;
  p.inv_freq = inv_freq;
  p.scaling = scaling;
  p.half = half;
  p.dim = D;
  p.tokens = T;
  const bool vec = half % 8 == 0 && D % 8 == 0 && q_stride % 8 == 0 && q_out_stride % 8 == 0 && k_stride % 8 == 0 &&
                   k_out_stride % 8 == 0 && aeg::aligned(q, 16) && aeg::aligned(k, 16) && aeg::aligned(q_out, 16) &&
                   aeg::aligned(k_out, 16);
  void (*kern)(const aeg::RotaryParams) =
      dtype == AEG_DTYPE_BF16 ? (vec ? aeg::rotary_kernel<__nv_bfloat16, 8> : aeg::rotary_kernel<__nv_bfloat16, 1>)
                              : (vec ? aeg::rotary_kernel<__half, 8> : aeg::rotary_kernel<__half, 1>);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(T, int64_t(aeg::num_sms()) * 8)));
  cfg.blockDim = dim3(aeg::kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AEG_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  AEG_CHECK_LAUNCH("rotary_multi_axis");
  aeg::note_launch(cfg.stream, false);
  return AEG_OK;
}
