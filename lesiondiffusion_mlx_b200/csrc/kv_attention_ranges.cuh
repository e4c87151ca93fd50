// Attention of a few query rows, each warp on an equal range of the cached
// tokens' tiles: the line of tiles, the ranges, and the join of the pairs that lie in
// several of them.  Shared by the 8-bit and the 4-bit cache's kernels, which
// describe the scheme.
#pragma once

#include <algorithm>

#include "host_common.h"
#include "kv_attention.cuh"

namespace ldb {
namespace {

constexpr int kWarps = 4;           // per CTA; they share nothing but the tiles' line
constexpr int kMaxBatch = 2048;
constexpr float kFloor = -1.0e30f;  // reference of a row that has seen nothing
constexpr int kHeadroom = 15;       // the largest weight is 2^15, within f16; the sum is kept without it

struct AttnParams {
  KvView c;
  const void* q;
  void* out;
  long long q_ld, q_batch, out_ld, out_batch;
  int queries, group, rows;  // rows = queries * group per key/value head
  int tile_rows, row_tiles;
  int causal, q_vec, out_vec;
  float scale_log2;
  int negate;      // the 4-bit kernel: scale_log2 is a magnitude, the queries are turned
  int warps;       // of the grid
  float* o_part;   // [warp][2][tile rows][D]
  float* ml_part;  // [warp][2][tile rows][2]
  // Pairs split over warps: (item, pair, first warp, warps, or 0 for a pair that
  // is whole), by pair where there are fewer pairs than warps, else by first warp.
  int4* open_part;
  int open_by_pair;
  unsigned int* status;
};

// ------------------------------------------------------------ division of the work

template <int TILE>
__device__ __forceinline__ int tiles_of(int tokens) {
  return (tokens + TILE - 1) / TILE;
}
// Positions of one pair of an item: START, then one per tile (none without tokens).
template <int TILE, int START>
__device__ __forceinline__ int places_of(int tokens) {
  return tokens == 0 ? 0 : START + tiles_of<TILE>(tokens);
}

// `total` positions in ranges of equal length, the first ones one longer.
struct Ranges {
  int per, extra;
  __device__ __forceinline__ Ranges(int total, int warps) : per(total / warps), extra(total % warps) {}
  __device__ __forceinline__ int begin(int w) const { return w * per + min(w, extra); }
  __device__ __forceinline__ int of(int u) const {
    const int head = extra * (per + 1);
    return u < head ? u / (per + 1) : extra + (u - head) / per;
  }
};

// First position of each item on the line, a scan over blocks of items; their
// number in s_base[batch].  All threads of the CTA.
template <int TILE, int START>
__device__ __forceinline__ void lay_out_line(const KvView& c, int pairs, int* s_base, unsigned int* status) {
  __shared__ int s_warp[kWarps];
  const int warp = warp_id(), lane = lane_id();
  int before = 0, next = static_cast<int>(threadIdx.x) < c.batch ? kv_length(c, threadIdx.x, status) : 0;
  for (int b0 = 0; b0 < c.batch; b0 += kWarps * 32) {
    const int b = b0 + threadIdx.x;
    const int n = b < c.batch ? places_of<TILE, START>(next) * pairs : 0;
    if (b + kWarps * 32 < c.batch) next = kv_length(c, b + kWarps * 32, status);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += s_warp[w];
    }
    if (b < c.batch) s_base[b] = before + upto - n;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) before += s_warp[w];
    __syncthreads();
  }
  if (threadIdx.x == 0) s_base[c.batch] = before;
  __syncthreads();
}

// Zeros for items without tokens, their rows dealt out over the CTAs.
template <typename T, int D>
__device__ __forceinline__ void clear_idle(const AttnParams& p, const int* s_base) {
  const int lane = lane_id();
  for (int b0 = 0; b0 < p.c.batch; b0 += 32) {
    const int mine = b0 + lane;
    uint32_t idle = __ballot_sync(0xffffffffu, mine < p.c.batch && s_base[mine + 1] == s_base[mine]);
    for (; idle; idle &= idle - 1) {
      const int b = b0 + __ffs(idle) - 1, width = p.c.kv_heads * p.group * D;
      for (int i = (blockIdx.x + b) % gridDim.x; i < p.queries; i += gridDim.x) {
        T* row = static_cast<T*>(p.out) + b * p.out_batch + i * p.out_ld;
        if (p.out_vec) {
          for (int d = threadIdx.x; d < width / 8; d += kWarps * 32)
            reinterpret_cast<uint4*>(row)[d] = make_uint4(0, 0, 0, 0);
        } else {
          for (int d = threadIdx.x; d < width; d += kWarps * 32) row[d] = from_f32<T>(0.f);
        }
      }
    }
  }
}

// ------------------------------------------------------------------ fragments

// D (16 x 8) += A (16 x 16) B (16 x 8), f16.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// W bytes (4, 8 or 16) at a 16-byte unit of a swizzled tile.
template <int W>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[W / 4]) {
  if constexpr (W == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (W == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// 16 bytes: the first `bytes` of them from src, then zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------ joining

// Row blockIdx.y of a pair whose tiles lie in several ranges: its parts, one
// per warp from the one that starts it.  The threads weigh the parts first (the
// references' maximum is order-free, the sums go through a fixed tree), then the
// block's groups of D / 4 threads, four channels each, add every k-th part in order, and
// the groups' sums are added in order.  Small blocks: most have nothing to do.
template <int D, typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) kv_attention_merge_kernel(const AttnParams p) {
  constexpr int kLanes = D / 4, kGroups = THREADS / kLanes;
  __shared__ float4 s_v[kGroups][kLanes];
  __shared__ float s_red[2][THREADS / 32], s_f[THREADS];
  pdl_begin();
  int4 at = p.open_part[blockIdx.x];
  if (p.open_by_pair && kv_length(p.c, blockIdx.x / (p.c.kv_heads * p.row_tiles), p.status) == 0)
    at.w = 0;  // not written
  const int first = at.z, count = at.w, r = blockIdx.y;
  const int row = (at.y % p.row_tiles) * p.tile_rows + r;
  if (count == 0 || row >= p.rows) return;
  const int head = at.y / p.row_tiles;
  const int group = threadIdx.x / kLanes, lane4 = threadIdx.x % kLanes;
  // slot 1 of the warp that starts the pair, slot 0 of those that go on with it
  auto part = [&](int i) { return (static_cast<long long>(first + i) * 2 + (i == 0 ? 1 : 0)) * p.tile_rows + r; };
  float m = -INFINITY;  // (no part is: a row that has seen nothing has its kernel's least reference)
  for (int i = threadIdx.x; i < count; i += THREADS) m = fmaxf(m, p.ml_part[part(i) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane_id() == 0) s_red[0][warp_id()] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) m = fmaxf(m, s_red[0][w]);
  float l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < count; i0 += THREADS) {
    if (i0) __syncthreads();  // the round before has read s_f
    const int i = i0 + threadIdx.x;
    if (i < count) {
      const float2 ml = *reinterpret_cast<const float2*>(p.ml_part + part(i) * 2);
      const float half = ex2_approx(0.5f * (ml.x - m));
      s_f[threadIdx.x] = half * half;
      l += kv_scaled(ml.y, half);
    }
    __syncthreads();
    const int n = min(count - i0, THREADS);
#pragma unroll 8
    for (int k = group; k < n; k += kGroups) {
      const float4 o = reinterpret_cast<const float4*>(p.o_part + part(i0 + k) * D)[lane4];
      const float f = s_f[k];
      v.x = fmaf(o.x, f, v.x), v.y = fmaf(o.y, f, v.y), v.z = fmaf(o.z, f, v.z), v.w = fmaf(o.w, f, v.w);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (lane_id() == 0) s_red[1][warp_id()] = l;
  s_v[group][lane4] = v;
  __syncthreads();
  if (static_cast<int>(threadIdx.x) >= D) return;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) l += s_red[1][w];
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) sum += reinterpret_cast<const float*>(s_v[k])[threadIdx.x];
  static_cast<T*>(p.out)[at.x * p.out_batch + (row / p.group) * p.out_ld +
                         (static_cast<long long>(head) * p.group + row % p.group) * D + threadIdx.x] =
      from_f32<T>(l == 0.f ? 0.f : sum * fp8_pow2(-kHeadroom) / l);
}

// Partial rows of every warp, and the pairs left open.
size_t workspace_bytes_of(int warps, int rows, int head_dim) {
  return static_cast<size_t>(warps) * (2ull * rows * (head_dim + 2) * sizeof(float) + sizeof(int4));
}

// The join of what the grid's warps (`tile` tokens a position) left open.
template <int D, typename T>
int launch_merge(cudaStream_t stream, const AttnParams& p, int tile) {
  if (p.open_by_pair) {
    const int pairs = p.c.batch * p.c.kv_heads * p.row_tiles;
    const dim3 grid(pairs, std::min(p.tile_rows, p.rows));
    // Parts of a pair, at most.  More threads add up many parts (32768 tokens, 8
    // rows: 22.2 us with 1024, 26.3 with 256; 4 heads of 64 14.6 and 23.3) and start later
    // (77 tokens, 24 rows: 13.2 and 10.7).
    const long long parts =
        std::min<long long>(p.warps / pairs, static_cast<long long>(p.c.width) * p.c.page / tile);
    if (parts >= 64)
      return launch_kernel(kv_attention_merge_kernel<D, T, 1024>, grid, dim3(1024), 0, stream,
                           "kv_attention merge launch", p);
    return launch_kernel(kv_attention_merge_kernel<D, T, 256>, grid, dim3(256), 0, stream,
                         "kv_attention merge launch", p);
  }
  return launch_kernel(kv_attention_merge_kernel<D, T, 256>, dim3(p.warps, std::min(p.tile_rows, p.rows)), dim3(256), 0,
                       stream, "kv_attention merge launch", p);
}

}  // namespace
}  // namespace ldb
