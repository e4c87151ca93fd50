// Product of 8-bit rows and an 8-bit weight on the block-scaled tensor-core
// path (tcgen05 kind::mxf8f6f4):
//
//   y[m, n] = act(sum_k a[m, k] w[n, k] 2^(ea[m, k/128] + ew[n/128, k/128])
//                 + bias[n] + residual[m, n])
//
// The scales are powers of two (E8M0), so the tensor core applies them inside
// the product, in FP32, and the accumulator stays in TMEM over the whole of K;
// an FP32 scale per 128 channels would have to leave TMEM for every K block and
// be applied in registers.  The hardware takes one scale byte per 32 elements
// of K: the four products of a 128-channel block name the same byte of the
// 32-bit scale word, and a word holds four consecutive blocks.
//
// One CTA per SM walks 128-row x BN-column tiles: warp 0 loads the code tiles
// (TMA, 128-byte swizzle), warps 2-3 write the scale words of each four blocks in
// the order that tcgen05.cp spreads over TMEM lanes, warp 1 issues scale
// copies and products, warps 4-11 drain the accumulator of one tile while the
// next is computed in the other (two warps per 32 rows, alternating 32-column
// chunks, staged in shared memory for TMA stores where the output allows them).
// Grids with fewer tiles than SMs cut K into ranges whose FP32 partial sums a
// second kernel adds in order.
//
// PAIR: two CTAs run one 256-row tile (cta_group::2), each staging its own rows
// and half of the weight columns: 30 KB a K block where one CTA alone moves 44
// KB for 128 x 224 outputs, in and out of shared memory at 128 bytes a cycle,
// which is what bounds it (704 cycles a K block against 448 of products).
//
// One B200: 8190 x 4096 x 4096 bf16 with a residual 122 us (2240 TFLOP/s, 1.34
// of the bf16 burst rate; tensor pipe 69 % active, 627 cycles for a K block's 448
// of products); 6400 x 256 -> 1024 with GELU 14.4 us, bound by the epilogue; one
// row times 8192 x 2048 8.2 us, the start of the pipeline (2.6 us of weight).

#include <algorithm>

#include "fp8.cuh"
#include "host_common.h"

namespace ldb {
namespace {

constexpr int kEpilogueWarps = 8;
constexpr int kThreads = (4 + kEpilogueWarps) * 32;
constexpr int kTileM = 128;
constexpr int kMaxStages = 8;
constexpr int kScaleStages = 4;                // ring of scale groups in shared memory
constexpr int kScaleBytes = 512 + 1024;        // A words, then up to 256 B words
constexpr int kMaxBn = 224;
constexpr int kStagingBytes = 4096;            // per epilogue warp: 32 x 32 outputs, twice for 16-bit ones
constexpr int kSmemBudget = 184 * 1024;        // code stages
constexpr int kTmemCols = 512;
static_assert(2 * kMaxBn + kScaleStages * 12 <= kTmemCols, "two accumulators and the scale sets");

struct MatmulParams {
  const uint8_t* a_scales;
  const uint8_t* w_scales;
  const float* bias;      // may be null
  const void* residual;   // may be null
  void* out;
  float* partial;         // split > 1: [split][m][n]
  long long a_scales_ld, w_scales_ld, res_ld, out_ld;
  int m, n, k;
  int pair, bn, stages, box_m;
  int tiles_m, tiles_n, split, kb_per_split;
  int act, out_dtype;
  int vec;       // out and residual rows allow 16-byte accesses and TMA stores
  int bias_vec;  // so does the bias
};

// Scale words of tile row `row` (128-channel blocks kb .. kb + 3) of A; blocks
// and rows outside the operand count as scale 1 (their codes are zero).
__device__ __forceinline__ uint32_t a_scale_word(const MatmulParams& p, int row, int kb, int kblocks) {
  if (row >= p.m) return 0x7F7F7F7Fu;
  const uint8_t* s = p.a_scales + row * p.a_scales_ld + kb;
  if (kb + 4 <= kblocks) return *reinterpret_cast<const uint32_t*>(s);
  uint32_t w = 0x7F7F7F7Fu;
  for (int j = 0; j < 4 && kb + j < kblocks; ++j)
    w = (w & ~(0xFFu << (8 * j))) | (static_cast<uint32_t>(s[j]) << (8 * j));
  return w;
}
// Tile and K range of work item i: rows vary fastest, so neighbouring CTAs
// share a weight tile.
struct Work {
  int row0, col0, kb0, kb1, split;
};
template <bool PAIR>
__device__ __forceinline__ Work work_item(const MatmulParams& p, int i, int kblocks, int rank) {
  Work w;
  const int tm = i % p.tiles_m;
  const int rest = i / p.tiles_m;
  w.split = rest % p.split;
  w.row0 = PAIR ? (2 * tm + rank) * kTileM : tm * kTileM;
  w.col0 = (rest / p.split) * p.bn;
  w.kb0 = w.split * p.kb_per_split;
  w.kb1 = min(kblocks, w.kb0 + p.kb_per_split);
  return w;
}

// Paired FP32 arithmetic (sm_100 f32x2 instructions).
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t both(float v) { return pack2(v, v); }

// 0.5 y (1 + erf(y / sqrt 2)) of two values, as 0.5 (y + |y|) - 0.5 |y| erfc(|y| /
// sqrt 2), which does not cancel, with erfc by formula 7.1.26 of Abramowitz and Stegun:
// ten operations a value.  The formula is within 1.5e-7 of erfc, so the result within
// 0.75e-7 |y|, as close as 1 + erf in FP32 comes; relative to the tail of negative
// values that is 5e-5 at -3 and 2e-3 at -5.  The factor of erfc stops at 8, where erfc is
// zero in FP32: +infinity times it would be a NaN (-infinity gives one, as in the
// first form).  With erff, and one warp per 32 rows, the epilogue of a short K took
// twice the time of everything else.
__device__ __forceinline__ void gelu2(float& y0, float& y1) {
  const uint64_t a = pack2(fabsf(y0), fabsf(y1));
  const uint64_t z = mul2(a, both(0.70710678118654752f));
  const uint64_t half = mul2(a, both(0.5f));
  float d0, d1, e0, e1, h0, h1;
  unpack2(fma2(z, both(0.3275911f), both(1.f)), d0, d1);
  const uint64_t t = pack2(rcp_approx(d0), rcp_approx(d1));
  uint64_t q = fma2(both(-1.061405429f), t, both(1.453152027f));
  q = fma2(q, t, both(-1.421413741f));
  q = fma2(q, t, both(0.284496736f));
  q = fma2(q, t, both(-0.254829592f));
  unpack2(mul2(mul2(z, z), both(-1.4426950408889634f)), e0, e1);
  q = mul2(mul2(q, t), pack2(ex2_approx(e0), ex2_approx(e1)));  // -erfc(z)
  unpack2(half, h0, h1);
  unpack2(fma2(pack2(fminf(h0, 8.f), fminf(h1, 8.f)), q, fma2(pack2(y0, y1), both(0.5f), half)), y0, y1);
}
__device__ __forceinline__ float gelu1(float y) {
  float other = 0.f;
  gelu2(y, other);
  return y;
}

// 32 columns of one output row before the rounding: bias, residual, activation
// (outputs and residuals that allow 16-byte accesses).
template <typename T>
__device__ __forceinline__ void finish32(const MatmulParams& p, int row, int col, float (&v)[32]) {
  const bool full = col + 32 <= p.n;
  if (p.bias) {
    if (full && p.bias_vec) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 b = reinterpret_cast<const float4*>(p.bias + col)[j];
        v[4 * j] += b.x, v[4 * j + 1] += b.y, v[4 * j + 2] += b.z, v[4 * j + 3] += b.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col + j < p.n) v[j] += p.bias[col + j];
    }
  }
  if (p.residual && row < p.m) {
    const T* r = static_cast<const T*>(p.residual) + row * p.res_ld + col;
    if (full) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float a[8];
        load8<T>(r + 8 * c, a);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * c + j] += a[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col + j < p.n) v[j] += to_f32<T>(r[j]);
    }
  }
  if (p.act == LDB_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) gelu2(v[j], v[j + 1]);
  }
}

// The same for outputs that allow no 16-byte accesses: 32 x 32 FP32 values staged
// in shared memory, a column per lane, so that a warp's accesses are one row
// each.  (A row per lane, value by value: 12983 x 358 -> 1961 took 253 us instead
// of 59; whole rows of 1960 columns take 27.)
template <typename T>
__device__ __forceinline__ void finish_rows(const MatmulParams& p, int split, int row0, int col,
                                            const uint8_t* staging) {
  const int lane = lane_id(), rows = min(32, p.m - row0);
  const int c = col + lane;
  const bool live = c < p.n;
  const bool last = p.split == 1;  // else a range's partial sums
  const float bias = last && p.bias && live ? p.bias[c] : 0.f;
  const T* res = static_cast<const T*>(p.residual) + (p.residual ? row0 * p.res_ld + c : 0);
  float* part = p.partial + (static_cast<long long>(split) * p.m + row0) * p.n + c;
  T* out = static_cast<T*>(p.out) + row0 * p.out_ld + c;
  T a[32];  // all rows' loads in flight together
  if (last && p.residual) {
#pragma unroll
    for (int u = 0; u < 32; ++u) a[u] = live && u < rows ? res[u * p.res_ld] : from_f32<T>(0.f);
  }
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 8) {
    if (r0 >= rows) break;
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = *reinterpret_cast<const float*>(staging + swizzle_offset((r0 + u) * 128 + lane * 4, 128));
    if (!last) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (live && r0 + u < rows) part[static_cast<long long>(r0 + u) * p.n] = v[u];
      continue;
    }
    if (p.bias) {
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] += bias;
    }
    if (p.residual) {
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] += to_f32<T>(a[r0 + u]);
    }
    if (p.act == LDB_ACT_GELU) {
#pragma unroll
      for (int u = 0; u < 8; u += 2) gelu2(v[u], v[u + 1]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (live && r0 + u < rows) out[(r0 + u) * p.out_ld] = from_f32<T>(v[u]);
  }
}

// WHOLE: 16-byte accesses to the rows of what is written (and the residual's).
template <typename T, bool PAIR, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_matmul_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap wmap,
                      const __grid_constant__ CUtensorMap omap, const MatmulParams p, unsigned int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int w_rows = PAIR ? p.bn / 2 : p.bn;  // weight columns this CTA stages
  const int stage_bytes = kTileM * 128 + w_rows * 128;
  uint8_t* s_scales = smem + p.stages * stage_bytes;
  uint8_t* s_out = s_scales + kScaleStages * kScaleBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_out + kEpilogueWarps * kStagingBytes);
  uint64_t* full = bars;                       // [kMaxStages] codes have landed
  uint64_t* empty = full + kMaxStages;         // [kMaxStages] the products have read them
  uint64_t* sf_full = empty + kMaxStages;      // [kScaleStages] scale words are written
  uint64_t* sf_empty = sf_full + kScaleStages; // [kScaleStages] the copy and the products have read them
  uint64_t* acc_full = sf_empty + kScaleStages;  // [2] a tile's products are done
  uint64_t* acc_empty = acc_full + 2;            // [2] the epilogue has drained it
  uint64_t* drain = acc_empty + 2;               // an aborting CTA's last products
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id();
  const int lane = lane_id();
  const int kblocks = (p.k + kFp8Block - 1) / kFp8Block;
  const int items = p.tiles_m * p.tiles_n * p.split;
  const int rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;
  const int item0 = PAIR ? blockIdx.x >> 1 : blockIdx.x, item_step = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kScaleStages; ++s) {
      mbar_init(&sf_full[s], PAIR ? 64 : 32);  // (a pair's barriers of arrival are the leader's)
      mbar_init(&sf_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&acc_full[t], 1);
      mbar_init(&acc_empty[t], PAIR ? 2 * kEpilogueWarps : kEpilogueWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&amap);
    tma_prefetch_desc(&wmap);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // both CTAs' barriers exist before any arrival from the other
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_begin();

  if (warp == 0) {
    // -------------------------------------------------------------- codes
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      int loads = 0;
      const uint32_t bytes = static_cast<uint32_t>(p.box_m + w_rows) * 128;
      bool ok = true;
      for (int i = item0; ok && i < items; i += item_step) {
        const Work w = work_item<PAIR>(p, i, kblocks, rank);
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!mbar_wait(&empty[st], ph ^ 1u, abort_flag, status)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + st * stage_bytes;
          if constexpr (PAIR) {
            // the loads of both CTAs complete on the leader's barrier, which counts both's bytes
            if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * bytes);
            const uint32_t bar = mapa_shared(smem_u32(&full[st]), 0);
            tma_load_2d_pair(sa, &amap, bar, kb * 128, w.row0);
            tma_load_2d_pair(sa + kTileM * 128, &wmap, bar, kb * 128, w.col0 + rank * w_rows);
          } else {
            mbar_arrive_expect_tx(&full[st], bytes);
            tma_load_2d(sa, &amap, &full[st], kb * 128, w.row0);
            tma_load_2d(sa + kTileM * 128, &wmap, &full[st], kb * 128, w.col0);
          }
          ++loads;
          if (++st == p.stages) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
      if (*abort_flag && rank == 0) {
        // Let the loads in flight land before the CTA gives up its shared memory
        // (a pair's CTAs give it up together).
        volatile int never = 0;
        for (int back = 1; back <= min(loads, p.stages); ++back) {
          const int l = loads - back;
          mbar_wait(&full[l % p.stages], static_cast<uint32_t>(l / p.stages) & 1u, &never, status);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    if (rank == 0) {  // (the leader's, with pairs)
      auto copy = [](uint32_t to, uint64_t desc) {
        if constexpr (PAIR) {
          tmem_copy_scales_pair(to, desc);
        } else {
          tmem_copy_scales(to, desc);
        }
      };
      auto product = [](uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t more) {
        if constexpr (PAIR) {
          umma_ss_mx8_pair(d, a, b, idesc, sa, sb, more);
        } else {
          umma_ss_mx8(d, a, b, idesc, sa, sb, more);
        }
      };
      auto commit = [](uint64_t* bar) {
        if constexpr (PAIR) {
          umma_commit_pair_warp(bar, 3);  // in both CTAs
        } else {
          umma_commit_warp(bar);
        }
      };
      // Scale words in TMEM: a set of columns per ring slot, behind the two accumulators.
      const int sfb_cols = 4 * ((p.bn + 127) / 128);
      const uint32_t sf_cols = 4 + sfb_cols;
      const uint32_t sf_base = tmem + kTmemCols - kScaleStages * sf_cols;
      int st = 0, sst = 0, tile = 0;
      uint32_t ph = 0, sph = 0;
      bool ok = true;
      for (int i = item0; ok && i < items; i += item_step, ++tile) {
        const Work w = work_item<PAIR>(p, i, kblocks, rank);
        const uint32_t acc = tmem + (tile & 1) * p.bn;
        ok = warp_wait(&acc_empty[tile & 1], (static_cast<uint32_t>(tile >> 1) & 1u) ^ 1u, abort_flag, status);
        if (!ok) break;
        tc_fence_after();
        for (int kb = w.kb0; ok && kb < w.kb1; kb += 4) {
          if (!warp_wait(&sf_full[sst], sph, abort_flag, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sfa = sf_base + sst * sf_cols;
          const uint32_t sfb = sfa + 4;
          const uint32_t s_addr = smem_u32(s_scales + sst * kScaleBytes);
          copy(sfa, make_smem_desc(s_addr, 0, 128, kSwizzleNone));
          for (int c = 0; c < sfb_cols / 4; ++c)
            copy(sfb + 4 * c, make_smem_desc(s_addr + 512 + 512 * c, 0, 128, kSwizzleNone));
          const int kend = min(w.kb1, kb + 4);
          for (int b = kb; b < kend; ++b) {
            if (!warp_wait(&full[st], ph, abort_flag, status)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a_addr = smem_u32(smem + st * stage_bytes);
            const uint32_t w_addr = a_addr + kTileM * 128;
            const uint32_t idesc = make_idesc_mx8(PAIR ? 2 * kTileM : kTileM, p.bn, static_cast<uint32_t>(b - kb));
#pragma unroll
            for (int q = 0; q < 4; ++q)
              product(acc, make_smem_desc(a_addr + q * 32, 16, 1024, kSwizzle128),
                      make_smem_desc(w_addr + q * 32, 16, 1024, kSwizzle128), idesc, sfa, sfb,
                      (b > w.kb0 || q > 0) ? 1u : 0u);
            commit(&empty[st]);
            if (++st == p.stages) {
              st = 0;
              ph ^= 1u;
            }
          }
          commit(&sf_empty[sst]);  // the copy and the products have read this slot
          if (++sst == kScaleStages) {
            sst = 0;
            sph ^= 1u;
          }
        }
        if (ok) commit(&acc_full[tile & 1]);
      }
      if (*abort_flag) {
        volatile int never = 0;
        if constexpr (PAIR) {
          umma_commit_pair_warp(drain, 1);
        } else {
          umma_commit_warp(drain);
        }
        mbar_wait(drain, 0, &never, status);
      }
    }
  } else if (warp < 4) {
    // -------------------------------------------------------------- scales
    // Warps 2 and 3 take the groups in turn, each with its next group's words
    // on their way while one's are written: with one warp their latency was
    // longer than the products of four blocks.
    int i = item0, kb = 0;
    Work w = work_item<PAIR>(p, min(i, items - 1), kblocks, rank);
    kb = w.kb0;
    auto advance = [&]() {  // to the next group
      kb += 4;
      if (kb >= w.kb1) {
        i += item_step;
        if (i < items) {
          w = work_item<PAIR>(p, i, kblocks, rank);
          kb = w.kb0;
        }
      }
    };
    uint32_t a[4], byte = 0x7F;
    // A tile's columns lie in at most three 128-column blocks: lane 4 n + j
    // reads byte j of block n's word.
    auto load = [&]() {
#pragma unroll
      for (int c = 0; c < 4; ++c) a[c] = a_scale_word(p, w.row0 + 32 * c + lane, kb, kblocks);
      const int block = w.col0 / kFp8Block + (lane >> 2), at = kb + (lane & 3);
      byte = lane < 12 && block * kFp8Block < p.n && at < kblocks ? p.w_scales[block * p.w_scales_ld + at] : 0x7F;
    };
    if (warp == 3 && i < items) advance();
    if (i < items) load();
    int sst = warp - 2;
    uint32_t sph = 0;
    while (i < items) {
      const int col = w.col0 % kFp8Block + lane;
      const uint4 rows = make_uint4(a[0], a[1], a[2], a[3]);
      uint32_t words[3];
#pragma unroll
      for (int n = 0; n < 3; ++n) {
        words[n] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) words[n] |= __shfl_sync(0xffffffffu, byte, 4 * n + j) << (8 * j);
      }
      advance();
      if (i < items) advance();
      if (i < items) load();
      uint32_t b[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int n = (col + 32 * c) / kFp8Block;
        b[c] = n == 0 ? words[0] : (n == 1 ? words[1] : words[2]);
      }
      if (!warp_wait(&sf_empty[sst], sph ^ 1u, abort_flag, status)) break;
      uint4* dst = reinterpret_cast<uint4*>(s_scales + sst * kScaleBytes);
      dst[lane] = rows;
      dst[32 + lane] = make_uint4(b[0], b[1], b[2], b[3]);
      if (p.bn > 128) dst[64 + lane] = make_uint4(b[4], b[5], b[6], b[7]);
      fence_proxy_async_smem();
      if constexpr (PAIR) {
        mbar_arrive_cluster(mapa_shared(smem_u32(&sf_full[sst]), 0));
      } else {
        mbar_arrive(&sf_full[sst]);
      }
      sst += 2;
      if (sst >= kScaleStages) {
        sst -= kScaleStages;
        sph ^= 1u;
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------- epilogue
    constexpr int kRowBytes = 32 * sizeof(T);            // of a staged chunk
    constexpr int kBuffers = kStagingBytes / (32 * kRowBytes);
    uint8_t* staging = s_out + (warp - 4) * kStagingBytes;
    const int quarter = warp & 3;
    int tile = 0, buffer = 0;
    for (int i = item0; i < items; i += item_step, ++tile) {
      const Work w = work_item<PAIR>(p, i, kblocks, rank);
      if (!warp_wait(&acc_full[tile & 1], static_cast<uint32_t>(tile >> 1) & 1u, abort_flag, status)) break;
      tc_fence_after();
      const int row0 = w.row0 + quarter * 32, row = row0 + lane;
      const uint32_t acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (tile & 1) * p.bn;
      const int cols = row0 < p.m ? min(p.bn, p.n - w.col0) : 0;
      for (int c = 32 * ((warp - 4) >> 2); c < cols; c += 64) {
        uint32_t r[32];
        tmem_ld32(acc + c, r);
        tmem_wait_ld();
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        const int col = w.col0 + c;
        if constexpr (!WHOLE) {
#pragma unroll
          for (int h = 0; h < 8; ++h)
            *reinterpret_cast<float4*>(staging + swizzle_offset(lane * 128 + h * 16, 128)) =
                make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
          __syncwarp();
          finish_rows<T>(p, w.split, row0, col, staging);
          __syncwarp();
        } else if (p.split > 1) {
          if (row < p.m) {
            float* o = p.partial + (static_cast<long long>(w.split) * p.m + row) * p.n + col;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (col + 4 * j < p.n)
                reinterpret_cast<float4*>(o)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        } else {
          finish32<T>(p, row, col, v);
          // the store before last (16-bit) or last (FP32) has read this buffer
          uint8_t* out = staging + buffer * 32 * kRowBytes;
          if (lane == 0) bulk_wait_group_read<kBuffers - 1>();
          __syncwarp();
#pragma unroll
          for (int h = 0; h < kRowBytes / 16; ++h) {
            constexpr int kPer = 16 / sizeof(T);
            uint4 packed;
            T* e = reinterpret_cast<T*>(&packed);
#pragma unroll
            for (int j = 0; j < kPer; ++j) e[j] = from_f32<T>(v[h * kPer + j]);
            *reinterpret_cast<uint4*>(out + swizzle_offset(lane * kRowBytes + h * 16, kRowBytes)) = packed;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&omap, out, col, row0);  // rows and columns outside the output are left out
            bulk_commit_group();
          }
          if (++buffer == kBuffers) buffer = 0;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) {
          mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[tile & 1]), 0));
        } else {
          mbar_arrive(&acc_empty[tile & 1]);
        }
      }
    }
    if (lane == 0) bulk_wait_group_all();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the leader's products read both CTAs' memory
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_dealloc_pair(tmem, kTmemCols);
    } else {
      tmem_dealloc(tmem, kTmemCols);
    }
  }
}

// Sum of the K ranges in their order, then the epilogue; one thread per value.
template <typename T>
__global__ void __launch_bounds__(256) fp8_matmul_reduce_kernel(const MatmulParams p) {
  pdl_begin();
  const long long total = static_cast<long long>(p.m) * p.n;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long row = i / p.n;
    const int col = static_cast<int>(i - row * p.n);
    float v = 0.f;
    for (int s = 0; s < p.split; ++s) v += p.partial[s * total + i];
    if (p.bias) v += p.bias[col];
    if (p.residual) v += to_f32<T>(static_cast<const T*>(p.residual)[row * p.res_ld + col]);
    if (p.act == LDB_ACT_GELU) v = gelu1(v);
    static_cast<T*>(p.out)[row * p.out_ld + col] = from_f32<T>(v);
  }
}

// Column tile, K ranges and ring depth from the extents alone.
int plan(int m, int n, int k, MatmulParams* p) {
  constexpr int kMost = 0x7FFFFE00;  // (rows and columns of a whole last tile still count in 32 bits)
  if (m <= 0 || n <= 0 || k <= 0 || m > kMost || n > kMost || k > kMost)
    return fail(LDB_ERR_SHAPE, "matmul_fp8: %d x %d x %d", m, n, k);
  const int sms = sm_count();
  const int kblocks = (k + kFp8Block - 1) / kFp8Block;
  p->m = m, p->n = n, p->k = k;
  // Cycles of a CTA that walks `waves` tiles.  A K block moves 128 rows of A and
  // its share of the weight through shared memory twice (in, and out to the tensor
  // core) at 128 bytes a cycle, and takes 2 cycles a column of products; the epilogue takes
  // about 32 cycles a column and runs beside the next tile's products.  K ranges
  // (few tiles, long K; cut at groups of four blocks) cost the second kernel, most of it
  // on the host; pairs start and end later.  Measured on one B200, us: 6400 x
  // 1024 x 1024 with residual 16.5 alone, 18.9 in pairs; 8190 x 4096 x 4096 156
  // alone, 125 in pairs; 6400 x 1024 x 256 with GELU 13.3 at 128 columns, 17.3 at 64, 14.9 at 224.
  long long best = -1;
  const int groups = (kblocks + 3) / 4;
  for (const int pair : {0, 1}) {
    if (pair && m <= kTileM) continue;
    const int tiles_m = (m + kTileM * (1 + pair) - 1) / (kTileM * (1 + pair));
    for (const int bn : {32, 64, 96, 128, 160, 192, kMaxBn}) {
      const int tiles_n = (n + bn - 1) / bn;
      const long long tiles = static_cast<long long>(tiles_m) * tiles_n;
      const int slots = pair ? sms / 2 : sms;
      int split = 1;
      if (!pair && tiles * 2 <= sms && kblocks >= 8)
        split = std::max(1, std::min({static_cast<int>(sms / tiles), groups, 16}));
      const int per = 4 * ((groups + split - 1) / split);
      split = (kblocks + per - 1) / per;
      const long long waves = (tiles * split + slots - 1) / slots;
      const long long main =
          static_cast<long long>(std::min(per, kblocks)) * (pair ? std::max(2 * bn, 256 + bn) : 256 + 2 * bn);
      const long long cost =
          waves * (std::max<long long>(main, 32 * bn) + 1000) + (split > 1 ? 6000 : 0) + (pair ? 5000 : 0);
      if (best < 0 || cost < best) {
        best = cost;
        p->pair = pair;
        p->bn = bn;
        p->tiles_m = tiles_m;
        p->tiles_n = tiles_n;
        p->split = split;
        p->kb_per_split = per;
      }
    }
  }
  const long long tiles = static_cast<long long>(p->tiles_m) * p->tiles_n;
  p->stages = std::min(kMaxStages, kSmemBudget / (kTileM * 128 + (p->pair ? p->bn / 2 : p->bn) * 128));
  p->box_m = std::min(kTileM, (m + 7) / 8 * 8);
  if (tiles * p->split > 0x7FFFFFFF) return fail(LDB_ERR_SHAPE, "matmul_fp8: too many tiles");
  return LDB_OK;
}

size_t partial_bytes(const MatmulParams& p) {
  return p.split > 1 ? static_cast<size_t>(p.split) * p.m * p.n * sizeof(float) : 0;
}

template <typename T, bool WHOLE>
int launch(cudaStream_t stream, const CUtensorMap& amap, const CUtensorMap& wmap, const MatmulParams& p,
           unsigned int* status) {
  static unsigned long long configured = 0;
  constexpr int kFixed = 1024 + kScaleStages * kScaleBytes + kEpilogueWarps * kStagingBytes + 512;
  static_assert(kFixed + kSmemBudget <= 232448, "shared memory");
  const int smem = kFixed + p.stages * (kTileM + (p.pair ? p.bn / 2 : p.bn)) * 128;
  CUtensorMap omap = amap;  // (not used without TMA stores)
  int rc = LDB_OK;
  if (WHOLE && p.split == 1) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.n), static_cast<uint64_t>(p.m)};
    const uint64_t strides[1] = {static_cast<uint64_t>(p.out_ld) * sizeof(T)};
    const uint32_t box[2] = {32, 32};
    if (sizeof(T) == 4) {
      rc = encode_tiled_f32(&omap, p.out, 2, dims, strides, box, 128);
    } else {
      rc = encode_tiled_f16(&omap, p.out, 2, dims, strides, box, 64, p.out_dtype == LDB_BF16);
    }
    if (rc != LDB_OK) return rc;
  }
  if (p.pair) {
    static unsigned long long pair_configured = 0;
    rc = ensure_smem_attribute(reinterpret_cast<const void*>(fp8_matmul_kernel<T, true, WHOLE>), kFixed + kSmemBudget,
                               &pair_configured, "matmul_fp8 shared memory");
    if (rc != LDB_OK) return rc;
    const int pairs = std::min(p.tiles_m * p.tiles_n, sm_count() / 2);
    return launch_kernel_cluster(fp8_matmul_kernel<T, true, WHOLE>, dim3(2 * pairs), dim3(kThreads), smem, stream,
                                 "matmul_fp8 (CTA pairs) launch", 2u, amap, wmap, omap, p, status);
  }
  rc = ensure_smem_attribute(reinterpret_cast<const void*>(fp8_matmul_kernel<T, false, WHOLE>), kFixed + kSmemBudget,
                             &configured, "matmul_fp8 shared memory");
  if (rc != LDB_OK) return rc;
  const int items = p.tiles_m * p.tiles_n * p.split;
  rc = launch_kernel(fp8_matmul_kernel<T, false, WHOLE>, dim3(std::min(items, sm_count())), dim3(kThreads), smem, stream,
                     "matmul_fp8 launch", amap, wmap, omap, p, status);
  if (rc != LDB_OK || p.split == 1) return rc;
  const long long total = static_cast<long long>(p.m) * p.n;
  const int blocks = static_cast<int>(std::min<long long>((total + 255) / 256, 4ll * sm_count()));
  return launch_kernel(fp8_matmul_reduce_kernel<T>, dim3(blocks), dim3(256), 0, stream, "matmul_fp8 reduce launch", p);
}

template <typename T>
int launch_rows(cudaStream_t stream, const CUtensorMap& amap, const CUtensorMap& wmap, const MatmulParams& p,
                unsigned int* status) {
  const bool whole = p.split > 1 ? p.n % 4 == 0 : p.vec != 0;
  return whole ? launch<T, true>(stream, amap, wmap, p, status) : launch<T, false>(stream, amap, wmap, p, status);
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_matmul_fp8_workspace_size(int m, int n, int k, size_t* bytes) {
  using namespace ldb;
  if (!bytes) return fail(LDB_ERR_INVALID, "matmul_fp8: bytes is null");
  MatmulParams p{};
  const int rc = plan(m, n, k, &p);
  if (rc == LDB_OK) *bytes = partial_bytes(p);
  return rc;
}

int ldb_matmul_fp8(cudaStream_t stream, const uint8_t* a, long long a_ld, const uint8_t* a_scales,
                   long long a_scales_ld, const uint8_t* w, long long w_ld, const uint8_t* w_scales,
                   long long w_scales_ld, const float* bias, const void* residual, long long residual_ld, void* out,
                   long long out_ld, int m, int n, int k, int act, int out_dtype, void* workspace,
                   size_t workspace_bytes) {
  using namespace ldb;
  if (!a || !a_scales || !w || !w_scales || !out) return fail(LDB_ERR_INVALID, "matmul_fp8: null pointer");
  if (out_dtype != LDB_F16 && out_dtype != LDB_F32 && out_dtype != LDB_BF16)
    return fail(LDB_ERR_INVALID, "matmul_fp8: unknown output type %d", out_dtype);
  if (act != LDB_ACT_NONE && act != LDB_ACT_GELU)
    return fail(LDB_ERR_INVALID, "matmul_fp8: unknown activation %d", act);
  MatmulParams p{};
  int rc = plan(m, n, k, &p);
  if (rc != LDB_OK) return rc;
  const int kblocks = (k + kFp8Block - 1) / kFp8Block;
  if (a_ld < k || w_ld < k || a_scales_ld < kblocks || w_scales_ld < kblocks || out_ld < n ||
      (residual && residual_ld < n))
    return fail(LDB_ERR_SHAPE, "matmul_fp8: a row stride is shorter than its row");
  if (a_ld % 16 || w_ld % 16 || reinterpret_cast<uintptr_t>(a) % 16 || reinterpret_cast<uintptr_t>(w) % 16)
    return fail(LDB_ERR_ALIGNMENT, "matmul_fp8: codes need 16-byte aligned rows");
  if (a_scales_ld % 4 || reinterpret_cast<uintptr_t>(a_scales) % 4)
    return fail(LDB_ERR_ALIGNMENT, "matmul_fp8: row scales need 4-byte aligned rows");
  const size_t need = partial_bytes(p);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(LDB_ERR_WORKSPACE, "matmul_fp8 needs %zu workspace bytes (16-byte aligned), got %zu", need,
                workspace_bytes);
  unsigned int* status = device_status_ptr();
  if (!status) return fail(LDB_ERR_CUDA, "matmul_fp8: no device status word");
  p.a_scales = a_scales, p.a_scales_ld = a_scales_ld;
  p.w_scales = w_scales, p.w_scales_ld = w_scales_ld;
  p.bias = bias, p.residual = residual, p.res_ld = residual_ld;
  p.out = out, p.out_ld = out_ld, p.partial = static_cast<float*>(workspace);
  p.act = act, p.out_dtype = out_dtype;
  const int es = out_dtype == LDB_F32 ? 4 : 2;
  p.vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_ld * es % 16 == 0 &&
          (!residual || (reinterpret_cast<uintptr_t>(residual) % 16 == 0 && residual_ld * es % 16 == 0));
  p.bias_vec = reinterpret_cast<uintptr_t>(bias) % 16 == 0;
  CUtensorMap amap, wmap;
  const uint64_t adims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(m)};
  const uint64_t wdims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(n)};
  const uint64_t astride[1] = {static_cast<uint64_t>(a_ld)}, wstride[1] = {static_cast<uint64_t>(w_ld)};
  const uint32_t abox[2] = {128, static_cast<uint32_t>(p.box_m)};
  const uint32_t wbox[2] = {128, static_cast<uint32_t>(p.pair ? p.bn / 2 : p.bn)};
  rc = encode_tiled_u8(&amap, a, 2, adims, astride, abox, 128);
  if (rc == LDB_OK) rc = encode_tiled_u8(&wmap, w, 2, wdims, wstride, wbox, 128);
  if (rc != LDB_OK) return rc;
  if (out_dtype == LDB_F16) return launch_rows<__half>(stream, amap, wmap, p, status);
  if (out_dtype == LDB_BF16) return launch_rows<__nv_bfloat16>(stream, amap, wmap, p, status);
  return launch_rows<float>(stream, amap, wmap, p, status);
}

}  // extern "C"
