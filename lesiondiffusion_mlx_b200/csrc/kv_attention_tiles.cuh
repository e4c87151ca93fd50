// Attention of many query rows over a paged cache, on the tcgen05 tensor cores: what
// the 8-bit and the 4-bit cache's kernels share.  A CTA owns two tiles of rows of one item and
// key/value head and streams blocks of tokens once for both; token ranges of a
// pair are merged in order by a second kernel.
#pragma once

#include <algorithm>

#include "host_common.h"
#include "kv_attention.cuh"
#include "packed.cuh"

namespace ldb {
namespace {

constexpr int kM = 128;      // rows per tile
constexpr int kN = 128;      // tokens per block
constexpr float kFloor = -1.0e30f;  // reference of a row that has seen nothing
constexpr float kGrow = 8.f;        // a reference follows its row's maximum once that is 2^8 above
constexpr int kHeadroom = 7;        // weights are 2^7 at the reference, 2^15 at most; the sum is kept without it

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Each lane writes 8 consecutive 32-bit columns of its own TMEM lane.
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// The CTA's share of the work.
struct Span {
  int b, head, row0, tiles, len, jb0, nblocks, open;
};
__device__ __forceinline__ Span span_of(const KvTileParams& p, unsigned int* status) {
  Span s;
  s.b = blockIdx.z;
  s.head = blockIdx.y;
  const int block = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
  s.row0 = (p.row_blocks - 1 - block) * 2 * kM;  // (causal: the rows that see most first)
  s.tiles = p.rows - s.row0 > kM ? 2 : 1;
  s.len = kv_length(p.c, s.b, status);
  const int last = min(p.rows, s.row0 + 2 * kM) - 1;
  const int seen = p.causal ? min(s.len, s.len - p.queries + last / p.group + 1) : s.len;
  const int blocks = seen > 0 ? (seen + kN - 1) / kN : 0;
  const int chunk = (blocks + p.splits - 1) / p.splits;
  s.jb0 = split * chunk;
  s.nblocks = max(0, min(blocks - s.jb0, chunk));
  s.open = p.causal ? min(s.len, s.len - p.queries + s.row0 / p.group + 1) : s.len;  // keys that every row sees
  return s;
}

// One warp per row: the ranges' parts in order.
template <int D, typename T>
__global__ void __launch_bounds__(256) kv_tiles_merge_kernel(const KvTileParams p) {
  pdl_begin();
  const long long total = static_cast<long long>(p.c.batch) * p.c.kv_heads * p.rows;
  const long long at = blockIdx.x * 8ll + warp_id();
  if (at >= total) return;
  const int lane = lane_id();
  float m = -INFINITY;  // (no part is: a row that has seen nothing has its kernel's least reference)
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.ml_part[(s * total + at) * 2]);
  float l = 0.f, v[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) v[c] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(p.ml_part + (s * total + at) * 2);
    const float half = ex2_approx(0.5f * (ml.x - m)), f = half * half;
    l += kv_scaled(ml.y, half);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) v[c] = fmaf(p.o_part[(s * total + at) * D + 32 * c + lane], f, v[c]);
  }
  const float inv = l == 0.f ? 0.f : fp8_pow2(-kHeadroom) / l;
  const long long pair = at / p.rows;
  const int row = static_cast<int>(at - pair * p.rows);
  const int head = static_cast<int>(pair % p.c.kv_heads);
  T* dst = static_cast<T*>(p.out) + (pair / p.c.kv_heads) * p.out_batch + (row / p.group) * p.out_ld +
           (static_cast<long long>(head) * p.group + row % p.group) * D;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) dst[32 * c + lane] = from_f32<T>(v[c] * inv);
}

// Ranges of tokens, from the table's capacity, in the time of a block of 128
// tokens: a CTA's start and end take about five, the partial rows are written
// and read once, and there is a second kernel; at most four waves.  The lengths are
// on the device: items much shorter than their table has columns get too many ranges, most of them
// empty, whose partial rows are written and read all the same (512 queries over 1000 tokens, 32
// heads of 128 over 8: 30 us in a table of 1024 tokens, 35 of 16384, 81 of 131072; over 8000
// tokens 99 of 8000 to 32000, 138 of 128000).  7 items of up to 19724 tokens, 523 causal queries, 4 heads of 32: 324 us in
// one range, 149 in five.
int kv_tile_splits(int batch, int kv_heads, long long rows, int head_dim, long long capacity) {
  const long long ctas = (rows + 2 * kM - 1) / (2 * kM) * kv_heads * batch, sms = sm_count();
  const long long blocks = (capacity + kN - 1) / kN;
  const long long most = std::min({32ll, 4 * sms / std::max(1ll, ctas), (blocks + 1) / 2});
  const double merge = static_cast<double>(batch) * kv_heads * rows * head_dim * 8 / 12e6;  // of a range
  double best = static_cast<double>((ctas + sms - 1) / sms) * (blocks + 5);
  int splits = 1;
  for (int s = 2; s <= most; ++s) {
    const double cost = static_cast<double>((ctas * s + sms - 1) / sms) * ((blocks + s - 1) / s + 5) + 2 + merge * s;
    if (cost < best) best = cost, splits = s;
  }
  return splits;
}

}  // namespace
}  // namespace ldb
