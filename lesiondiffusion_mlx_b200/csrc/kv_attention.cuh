// What the two cache-attention kernels share: the split of a query into e4m3
// parts, the NaN tests of packed codes, and the many-row kernel's interface.
#pragma once

#include <type_traits>

#include "host_common.h"
#include "kv_cache.cuh"

namespace ldb {

// Four values as e4m3, and what is left of them (exact) times SCALE: the next part's input.
template <int SCALE>
__device__ __forceinline__ uint32_t kv_split_part(__half2 (&x)[2]) {
  uint32_t codes = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint16_t part;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(part) : "r"(*reinterpret_cast<const uint32_t*>(&x[h])));
    const uint32_t back = fp8_unpack2(part);
    x[h] = __hsub2(x[h], *reinterpret_cast<const __half2*>(&back));
    if (SCALE != 1) x[h] = __hmul2(x[h], __float2half2_rn(static_cast<float>(SCALE)));
    codes |= static_cast<uint32_t>(part) << (16 * h);
  }
  return codes;
}

template <typename T>
__device__ __forceinline__ float2 kv_unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

// Non-zero if one of four codes is a NaN (0x7F or 0xFF).
__device__ __forceinline__ uint32_t kv_nan_codes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// The same codes with each NaN turned into zero.
__device__ __forceinline__ uint32_t kv_without_nan(uint32_t w) { return w & ~((kv_nan_codes(w) >> 7) * 0xFFu); }

// The power of two of a row's largest magnitude, within what its factors can express.
__device__ __forceinline__ int kv_query_exponent(float m) {
  return m > 0.f ? min(126, max(-119, static_cast<int>(__float_as_uint(m) >> 23) - 127)) : 0;
}

// A softmax sum adds up 2^(s - M) with M the maximum of s + ev, as the weight
// 2^(s + ev - M) times 2^-ev.  That weight is zero in FP32 from 2^-126 on, although the
// term still counts, where a page's exponent lies far below that of the page
// that sets M: such pages' terms are computed apart, without ev.  For the others
// what is lost is below 2^(kKvFar - 126) of a term that the sum has.
constexpr float kKvFar = 64.f;
__device__ __forceinline__ bool kv_far_below(float ev, float top) { return ev < top - kKvFar && ev >= -127.f; }

// sum 2^x for x <= 0 that may lie below FP32's range while the result does not: in two halves.
__device__ __forceinline__ float kv_scaled(float sum, float half) { return sum * half * half; }

struct KvTileParams {
  KvView c;
  const void* q;
  void* out;
  long long q_ld, q_batch, out_ld, out_batch;
  int queries, group, rows;  // rows = queries * group per key/value head
  int row_blocks, splits;
  int causal, q_vec, out_vec, negate;
  float scale_log2;  // magnitude; `negate` turns the queries
  float* o_part;     // [split][batch][kv head][row][D]
  float* ml_part;    // [split][batch][kv head][row][2]
};

// The many-row kernel (p's shapes and pointers filled in), and the bytes of the
// partial rows of its ranges for a table of `capacity` tokens (negative: any).
size_t kv_tile_workspace(int batch, int kv_heads, long long rows, int head_dim, long long capacity);
int kv_attention_tiles(cudaStream_t stream, KvTileParams p, int head_dim, int dtype, float scale, void* workspace,
                       unsigned int* status);

}  // namespace ldb
