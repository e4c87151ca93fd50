// The 8-bit format shared by the quantizing norm, the product and the
// key/value cache: e4m3 codes with one power-of-two scale (E8M0: a byte that
// stands for 2^(byte - 127)) per block of values.
//
// The scale of a block is the smallest 2^e with max|y| <= 448 * 2^e (448 is the
// largest e4m3 value), so y * 2^-e never saturates and the multiplication is
// exact: a code differs from y 2^-e by its own rounding (to nearest, ties to
// even) alone.  Values that are not finite are left out of the maximum and
// become the NaN code.  A block of zeros has the scale 1.
#pragma once

#include "common.cuh"

namespace ldb {

constexpr int kFp8Block = 128;  // channels per scale (and rows per scale of a weight)

// e with max|y| <= 448 * 2^e for a finite amax >= 0, from the bits of amax:
// amax = m 2^k, m in [1, 2), and 448 = 1.75 * 2^8.  FP32 subnormals count as
// the smallest normal (their e is below the E8M0 range either way).
__device__ __forceinline__ int fp8_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int k = static_cast<int>(bits >> 23) - 127;
  const int e = k - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return amax == 0.f ? 0 : max(e, -127);
}

// 2^e for e in [-127, 127] (2^-127 is an FP32 subnormal).
__device__ __forceinline__ float fp8_pow2(int e) {
  return __uint_as_float(e > -127 ? static_cast<uint32_t>(e + 127) << 23 : 0x00400000u);
}

// Two values to e4m3, rounded to nearest even: lo in the low byte.  NaN
// becomes the NaN code; magnitudes past 448 (infinities too) saturate, so
// callers turn infinities into NaN first.
__device__ __forceinline__ uint32_t fp8_pack2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  return fp8_pack2(a, b) | (fp8_pack2(c, d) << 16);
}

// Two codes (low byte first) to packed f16: exact, NaN codes stay NaN.
__device__ __forceinline__ uint32_t fp8_unpack2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
  return r;
}

__device__ __forceinline__ bool fp8_is_finite(float v) { return fabsf(v) < __uint_as_float(0x7F800000u); }
__device__ __forceinline__ float fp8_nan() { return __uint_as_float(0x7FC00000u); }

// Element types of the 16- and 32-bit sides.
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}

// Eight consecutive elements to / from FP32, as 16-byte accesses (p aligned).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0];
    const float4 b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
}

}  // namespace ldb
