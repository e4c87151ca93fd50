// What the 4-bit cache's attention kernels share.
#pragma once

#include "kv_attention.cuh"

namespace ldb {

// A row's reference M is the rounded product of a score and the row's factor, and a weight's exponent fma(s, factor,
// headroom - M).  Past 2^20 the rounding of M and of headroom - M is not small against the exponent (from 2^24 on it is
// a whole power of two, and weights overflow or vanish): from there on a score is rounded as M is before M is taken
// off, so that the largest meets it exactly.
constexpr float kFarReference = 1048576.f;
// The reference of a row that has seen nothing: below every score that is finite by a factor of 1.1.
constexpr float kUnseen = -3.0e38f;
__device__ __forceinline__ bool is_far(float reference) {
  return fabsf(reference) > kFarReference && reference != kUnseen;
}

// The many-row kernel (p's shapes and pointers filled in), and the
// bytes of the partial rows of its ranges for a table of `capacity` tokens.
size_t kv_int4_tile_workspace(int batch, int kv_heads, long long rows, int head_dim, long long capacity);
int kv_int4_attention_tiles(cudaStream_t stream, KvTileParams p, int head_dim, int dtype, float scale, void* workspace,
                            unsigned int* status);

}  // namespace ldb
