// The 4-bit format of the paged key/value cache.
//
// A token's channels come in groups of 16 with one scale each:
//
//   value = (code - 8) s,   code in 0 .. 15
//
// s has five bits of exponent and three of mantissa: its byte is an f16's upper eight
// bits under the sign, so s is one shift away from an f16 and (code - 8) s is
// exact in f16, bf16 and FP32.  Quantizing takes the least s with max|x| <= 7.5 s:
// then no value is further than s / 2 from its code's (7.5 s goes to 7 s, -7.5 s to -8 s).
// Bytes above kInt4TopScale are not used but for 255, a NaN, the scale of a group that holds a
// value that is not finite.
//
// Codes are packed two to a byte, the lower channel in the low half:
// codes[page][kv head][token in page][D / 2]; scales lie token by token within a
// group, scales[page][kv head][D / 16][token in page], so that a group's scales of
// neighbouring tokens are one word.
//
// (Groups of 16 normal values keep 21.4 dB of signal to error so; the 4-bit floating
// point codes 0, 0.5, 1, 1.5, 2, 3, 4, 6 with the same scales keep 20.0.)
#pragma once

#include "fp8.cuh"
#include "packed.cuh"

namespace ldb {

constexpr int kInt4Group = 16;     // channels per scale
constexpr int kInt4TopScale = 198; // 1.75 * 2^9: 72 times it is within f16 (kernels take codes as 64 + code)
constexpr int kInt4NanScale = 255;
constexpr int kInt4Quad = 4;       // tokens whose scales are one word

__device__ __forceinline__ float int4_scale_value(int byte) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(byte << 7)));
}

// The byte of the least scale with amax <= 7.5 s, for a finite amax >= 0: the
// quotient's leading bits, and one more where they fall short (7.5 s is exact;
// the quotient's own rounding may cost a second step for FP32 inputs).
__device__ __forceinline__ int int4_scale_byte(float amax) {
  const float t = amax * (1.f / 7.5f);
  int byte = t < 6.103515625e-05f ? static_cast<int>(t * 131072.f)
                                  : static_cast<int>(__float_as_uint(t) >> 20) - ((127 - 15) << 3);
  byte = min(byte, kInt4TopScale);
#pragma unroll
  for (int n = 0; n < 2; ++n)
    if (byte < kInt4TopScale && 7.5f * int4_scale_value(byte) < amax) ++byte;
  return byte;
}

// 1 / s in two parts: x / s to within 2^-46, so that ties (frequent among 16-bit
// values) are met exactly and go to the even code.
struct Int4Inverse {
  float hi, lo;
  __device__ __forceinline__ explicit Int4Inverse(int byte) {
    const float s = int4_scale_value(byte);
    hi = __frcp_rn(s);
    lo = hi * fmaf(-s, hi, 1.f);
    if (byte == 0 || byte == kInt4NanScale) hi = lo = 0.f;
  }
};

// Eight values (pairs of neighbours) within -8.5 s .. 7.5 s to packed codes.
__device__ __forceinline__ uint32_t int4_pack8(const uint64_t (&x)[4], const Int4Inverse& inv) {
  // Adding 1.5 * 2^23 rounds to the nearest integer, which the sum's low bits then hold.
  constexpr uint32_t kBias = 0x4B400000u, kOnes = 0x11111111u;
  constexpr float kMagic = 12582912.f + 8.f;
  const uint64_t hi = pack2(inv.hi, inv.hi), lo = pack2(inv.lo, inv.lo), magic = pack2(kMagic, kMagic);
  uint32_t word = 0;
#pragma unroll
  for (int k = 3; k >= 0; --k) {
    float a, b;
    unpack2(fma2(x[k], hi, mul2(x[k], lo)), a, b);
    unpack2(add2(pack2(fminf(a, 7.f), fminf(b, 7.f)), magic), a, b);
    word = (word * 16u + __float_as_uint(b)) * 16u + __float_as_uint(a);
  }
  return word - kBias * kOnes;
}

// ------------------------------------------------------------ unpacking to f16

__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ uint32_t as_word(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// The scale bytes of `word` that `sel` names (the lower and the upper one as f16, see scale_selector).
__device__ __forceinline__ uint32_t scale_pair(uint32_t word, uint32_t sel) { return __byte_perm(word, 0, sel) * 128u; }
__device__ __forceinline__ uint32_t scale_selector(int lower, int upper) { return 0x4040u | lower | upper << 8; }

// (a & mask) | bits in one instruction (as plain C, with two constants, it became two).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
  return d;
}

// The four pairs of codes (n, n + 4) of a word's two halves as values.  A code in bits 4 .. 7 of an f16
// whose upper bits are those of 64 is 64 + code: (64 + code) s - 72 s, exactly.  In bits 0 .. 3 under 1024
// it is 1024 + code, and 1032 s may be past f16's range: 1032 is taken off first.  (Both at bits 4 .. 7 takes two
// more shifts and two fewer subtractions: as many instructions, but of the integer pipe, which is the busier: 262144
// tokens 71.1 us so, 69.3 as here.)
__device__ __forceinline__ void unpack4(uint32_t w, __half2 s, __half2 minus72s, uint32_t (&v)[4]) {
  constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u, k64 = 0x54005400u, k1024 = 0x64006400u;
  const __half2 minus1032 = __float2half2_rn(-1032.f);
  const uint32_t u = w >> 8;
  v[0] = as_word(__hmul2(__hadd2(as_half2(and_or(w, kLow, k1024)), minus1032), s));
  v[1] = as_word(__hfma2(as_half2(and_or(w, kHigh, k64)), s, minus72s));
  v[2] = as_word(__hmul2(__hadd2(as_half2(and_or(u, kLow, k1024)), minus1032), s));
  v[3] = as_word(__hfma2(as_half2(and_or(u, kHigh, k64)), s, minus72s));
}
__device__ __forceinline__ __half2 minus72(uint32_t s) { return __hmul2(as_half2(s), __float2half2_rn(-72.f)); }

}  // namespace ldb
