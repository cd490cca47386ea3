// The 4-bit KV-cache tile: 16 tokens of one (block, layer, KV head), 128 dims, keys and values.
//
// An element stands for code * scale + minimum, with one (scale, minimum) pair of the model's
// 16-bit type per token and 64-dim group:
//   minimum = min of the group (exact: it is one of the inputs)
//   scale   = (max - min) / 15, rounded once to the type (nearest, ties to even)
//   code    = (x - minimum) / scale, rounded to the nearest whole number (ties to even), 0..15
// A group whose max - min is not finite (a NaN, an infinity, or a spread beyond fp32) has NaN for
// both, so that it reads back as NaN instead of as plausible numbers; scale 0 has code 0.
//
// Bytes of a tile (2304 = 18 x 128, contiguous, so that one bulk copy fetches it):
//   [0, 1024)     key codes: token t at t * 64, in four 16-byte chunks; chunk c, word w holds dims
//                 32 w + 8 c + n at bits 4 n. Lane (row g, column c) of an MMA fragment finds all
//                 of its codes of token g in one 16-byte load, and words 0, 1 / 2, 3 belong to
//                 groups 0 / 1.
//   [1024, 2048)  value codes: tokens 2 p and 2 p + 1 at p * 128, in eight 16-byte chunks; chunk g,
//                 word w holds dims 64 (w / 2) + 8 g + 4 (w % 2) + n of token 2 p at bits 4 n and of
//                 token 2 p + 1 at bits 16 + 4 n. A byte belongs to one token, so writing a token
//                 touches no other one's bytes.
//   [2048, 2176)  key pairs: (scale, minimum) of token t, group g at t * 8 + g * 4
//   [2176, 2304)  value pairs, likewise
#pragma once

#include "aeg_common.cuh"

#include <type_traits>

namespace aeg {

constexpr int kInt4Dim = 128;
constexpr int kInt4Group = 64;
constexpr int kInt4TileBytes = 2304;
constexpr int kInt4TileElems = kInt4TileBytes / 2;
constexpr int kInt4ValueCodes = 1024;
constexpr int kInt4KeyPairs = 2048;
constexpr int kInt4ValuePairs = 2176;

// Byte offset of the key word that holds dims 8 l .. 8 l + 7 (l = 0..15) of token t.
__host__ __device__ __forceinline__ int int4_key_word(int t, int l) { return t * 64 + (l & 3) * 16 + (l >> 2) * 4; }
// Byte offset of the 16-bit half that holds value dims 8 l .. 8 l + 3 of token t; the half of dims
// 8 l + 4 .. 8 l + 7 lies 4 bytes further on.
__host__ __device__ __forceinline__ int int4_value_half(int t, int l) {
  return kInt4ValueCodes + (t >> 1) * 128 + (l & 7) * 16 + (l >> 3) * 8 + (t & 1) * 2;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The 16 bits of `v` rounded once to T: to 24 bits with the lost part kept as a sticky last bit
// (round to odd), from which the rounding to T's 8 or 11 bits comes out as if made from `v`.
template <typename T>
__device__ __forceinline__ T round_once(double v) {
  const float f = __double2float_rz(v);
  uint32_t bits = __float_as_uint(f);
  if (static_cast<double>(f) != v) bits |= 1u;
  return from_float<T>(__uint_as_float(bits));
}

template <typename T>
__device__ __forceinline__ uint32_t bits16(T v) {
  return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&v));
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// A scale rounded as if from infinite precision, for an exact span well within fp32's range: the quotient
// span / 15 by the rounded 1 / 15 and one correction is the nearest of 24 bits, the sign of its exact
// remainder says on which side of it the true one lies, and rounding that to odd (cut off, with a sticky
// last bit) leaves T's rounding as if made from the true quotient.
template <typename T>
__device__ __forceinline__ T scale_of_exact(float span) {
  constexpr float kFifteenth = 1.f / 15.f;
  const float q0 = span * kFifteenth;
  const float q = fmaf(fmaf(-15.f, q0, span), kFifteenth, q0);
  const float rest = fmaf(-15.f, q, span);
  uint32_t bits = __float_as_uint(q) - (rest < 0.f ? 1u : 0u);
  if (rest != 0.f) bits |= 1u;
  return from_float<T>(__uint_as_float(bits));
}

// 1 / s rounded to nearest, for a value s of T: one Newton step from the approximate reciprocal. With 8 or 11
// significant bits in s that is the rounded one from any start within 2 ulp (tried for every mantissa).
__device__ __forceinline__ float reciprocal_of_t(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return fmaf(r, fmaf(-s, r, 1.f), r);
}

// A lane's 8 elements.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float2 f = unpack2<T>(w[n]);
    x[2 * n] = f.x;
    x[2 * n + 1] = f.y;
  }
}

__device__ __forceinline__ uint32_t pair_of(uint32_t scale, uint32_t lo) { return scale | (lo << 16); }

// The general form of int4_quantise, right for every group. Codes: c = rint(d / s) by a reciprocal is
// right or next to it, c * s has at most 15 bits, and d - c * s comes out of one FMA exactly, as
// |d - c s| <= s and d <= 16 s or so. Only where it is exactly half a scale does the rounding error e of
// d = x - minimum itself count.
template <typename T>
__device__ __noinline__ uint2 int4_quantise_any(uint4 raw, float lo, float hi) {
  float x[8];
  unpack8<T>(raw, x);
  const bool ok = isfinite(hi - lo);
  const T scale = round_once<T>(ok ? (static_cast<double>(hi) - static_cast<double>(lo)) / 15.0 : 0.0);
  float s = to_float<T>(scale);
  uint32_t word = 0;
  const uint32_t pair = ok ? pair_of(bits16(scale), bits16(from_float<T>(lo))) : 0x7fff7fffu;
  if (!ok || s == 0.f) return make_uint2(0u, pair);
  // Far below 1, both sides are scaled up exactly so that the reciprocal stays finite.
  const float up = s < 1e-30f ? 18446744073709551616.f : 1.f;
  s *= up;
  const float r = __frcp_rn(s), half = 0.5f * s;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const float d0 = x[n] - lo, d = d0 * up;
    float c = fminf(rintf(d * r), 15.f);
    const float rest = fmaf(-c, s, d);
    if (fabsf(rest) >= half) {
      const float back = d0 - x[n];
      const float e = (x[n] - (d0 - back)) + (-lo - back);  // x - lo = d0 + e
      const bool odd = (static_cast<int>(c) & 1) != 0;
      if (rest > half || (rest == half && (e > 0.f || (e == 0.f && odd)))) c = fminf(c + 1.f, 15.f);
      else if (rest < -half || (rest == -half && (e < 0.f || (e == 0.f && odd)))) c -= 1.f;
    }
    word |= static_cast<uint32_t>(static_cast<int>(c)) << (4 * n);
  }
  return make_uint2(word, pair);
}

// Codes of a lane's 8 dims and its group's pair: {codes, dim n's at bits 4 n; scale | minimum << 16}. The
// 8 lanes of a group are consecutive; the whole warp calls this together.
//
// Where no element is below 2^(p - 23) of the span (p: T's significant bits; an exact 0 is taken for one, too),
// every x - minimum is a multiple of 2^-23 of the span or more. Then differences are exact in fp32, a quotient that is no tie
// differs from one by more than fp32's rounding, and a correctly rounded quotient gives the right code:
// that is a product and two FMAs (Markstein's division with the rounded reciprocal), and adding 1.5 * 2^23
// rounds it to a whole number, ties to even, with the code in the low bits. fp16 has no bits below 2^-24,
// so any group with a span below 1/2 is fine too. Groups that are not sure of it, with subnormal scales
// or without a finite span take the general form, with their warp. Writing a prompt batch of 11,348
// tokens x 4 heads took 21.7 us with the general form alone.
template <typename T>
__device__ __forceinline__ uint2 int4_quantise(const uint4& raw) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr float kLeast = kHalf ? 0x1p-12f : 0x1p-15f;
  constexpr float kNormal = kHalf ? 0x1p-14f : 1e-30f;  // least scale of the short form
  float x[8];
  unpack8<T>(raw, x);
  float lo = x[0], hi = x[0], least = fabsf(x[0]);
#pragma unroll
  for (int n = 1; n < 8; ++n) {
    lo = min_nan(lo, x[n]);
    hi = max_nan(hi, x[n]);
    least = fminf(least, fabsf(x[n]));
  }
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, off));
  }
  const float span = hi - lo;
  const bool sure = (least > span * kLeast || (kHalf && span < 0.5f)) && span > 16.f * kNormal && span < 3e38f;
  if (!__all_sync(0xffffffffu, sure)) return int4_quantise_any<T>(raw, lo, hi);
  const T scale = scale_of_exact<T>(span);
  const float s = to_float<T>(scale), r = reciprocal_of_t(s);
  uint32_t word = 0;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const float d = x[n] - lo, q0 = d * r;
    const float q = fmaf(fmaf(-q0, s, d), r, q0);
    word += (__float_as_uint(q + 12582912.f) & 15u) << (4 * n);
  }
  return make_uint2(word, pair_of(bits16(scale), bits16(from_float<T>(lo))));
}

}  // namespace aeg
