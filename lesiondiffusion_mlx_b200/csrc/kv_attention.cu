// Attention of a few query rows over the paged 8-bit key/value cache.
//
//   s[r, j] = (q_r . k_j) 2^ek scale        over the codes of key j's page
//   o_r = sum_j 2^(s - M) 2^ev v_j / sum_j 2^(s - M)     (s in log2 units)
//
// with one running reference per row, M = max_j (s[r, j] + ev_j), so that every
// weight 2^(s + ev - M) of the value product lies in [0, 1] whatever the
// pages' scales are, and is rounded to f16 once; the sum takes the same weight
// times 2^-ev in FP32.  Codes are exact in f16; bf16 queries become f16 after
// a power-of-two scaling of their row.
//
// Bound: HBM, the cached tokens (2 D bytes each) read once for a group's
// heads.  The 16 rows of an m16n8k16 product are (query, head of the group)
// pairs of one key/value head.  The cached tokens of all items and heads form one line of
// 64-token tiles, cut into equal ranges, one per CTA (two CTAs per SM), so that
// ragged lengths and preallocated tables leave no SM idle; a pair whose tiles
// lie in several CTAs is merged by a second kernel, in order.  One warp fetches tiles (TMA,
// swizzled) into a ring; four warps take them in turn, each with its own M, sum
// and output, merged at the end of a pair.  A lane's 16-byte reads of a
// swizzled row are free of bank conflicts, and the orders of channels (in q k)
// and of output columns (in p v) are chosen so that these bytes are its
// fragments.

#include <algorithm>

#include "host_common.h"
#include "kv_cache.cuh"

namespace ldb {
namespace {

constexpr int kTile = 64;        // tokens per tile
constexpr int kRows = 16;        // query rows of a product
constexpr int kConsumers = 4;    // warps that take tiles in turn
constexpr int kAttnThreads = (kConsumers + 1) * 32;
constexpr int kMaxBatch = 2048;
constexpr int kCtasPerSm = 2;
constexpr float kFloor = -1.0e30f;  // reference of a row that has seen nothing

struct AttnParams {
  KvView c;
  const void* q;
  void* out;
  long long q_ld, q_batch, out_ld, out_batch;
  int queries, group, rows, row_tiles;  // rows = queries * group per key/value head
  int causal, q_vec;
  float scale_log2;
  int ctas;
  float* o_part;   // [cta][2][16][D]
  float* ml_part;  // [cta][2][16][2]
};

template <int D>
struct Cfg {
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = D == 128 ? 4 : (D == 64 ? 6 : 8);
  static constexpr int kOffMeta = kStages * kStageBytes;            // [stage][4] (key factor, value exponent)
  static constexpr int kOffO = kOffMeta + kStages * 4 * 8;          // [4][16][D] floats
  static constexpr int kOffMl = kOffO + kConsumers * kRows * D * 4; // [4][16][2] floats
  static constexpr int kOffBar = kOffMl + kConsumers * kRows * 8;
  static constexpr int kOffBase = kOffBar + 2 * kStages * 8 + 16;   // [batch + 1] long long
};

// ------------------------------------------------------------ division of the work

__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + kTile - 1) / kTile; }

// CTAs that share `total` tiles: at least one tile per consumer warp.
__device__ __forceinline__ long long active_ctas(long long total, int ctas) {
  return max(1ll, min(static_cast<long long>(ctas), (total + kConsumers - 1) / kConsumers));
}
__device__ __forceinline__ long long range_begin(long long cta, long long total, long long active) {
  return cta * total / active;
}

struct Segment {
  int b, pair, tile0, tiles, item_tiles;
  bool whole;
};

// The segment that starts at tile u of the line (base: each item's first tile).
__device__ __forceinline__ Segment segment_at(const long long* base, int batch, int pairs, long long u, long long end) {
  int lo = 0, hi = batch;  // the last item whose first tile is at or before u
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (base[mid] <= u) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  Segment g;
  g.b = lo;
  const long long rel = u - base[lo];
  g.item_tiles = static_cast<int>((base[lo + 1] - base[lo]) / pairs);
  g.pair = static_cast<int>(rel / g.item_tiles);
  g.tile0 = static_cast<int>(rel - static_cast<long long>(g.pair) * g.item_tiles);
  g.tiles = static_cast<int>(min(static_cast<long long>(g.item_tiles - g.tile0), end - u));
  g.whole = g.tiles == g.item_tiles;
  return g;
}

// ------------------------------------------------------------------ fragments

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

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

template <int D, typename T>
__global__ void __launch_bounds__(kAttnThreads, kCtasPerSm)
    kv_attention_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const AttnParams p, unsigned int* status) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float2* s_meta = reinterpret_cast<float2*>(smem + C::kOffMeta);
  float* s_o = reinterpret_cast<float*>(smem + C::kOffO);
  float* s_ml = reinterpret_cast<float*>(smem + C::kOffMl);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + C::kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + C::kStages);
  long long* s_base = reinterpret_cast<long long*>(smem + C::kOffBase);
  const int warp = warp_id(), lane = lane_id();

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    *abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  pdl_begin();
  const int pairs = p.c.kv_heads * p.row_tiles;
  if (warp == 0) {
    // First tile of each item on the line.
    long long sum = 0;
    for (int b0 = 0; b0 < p.c.batch; b0 += 32) {
      const int b = b0 + lane;
      long long n = b < p.c.batch ? static_cast<long long>(tiles_of(kv_length(p.c, b, status))) * pairs : 0;
      long long upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
      }
      if (b < p.c.batch) s_base[b] = sum + upto - n;
      sum += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) s_base[p.c.batch] = sum;
  }
  __syncthreads();
  const long long total = s_base[p.c.batch];
  const long long active = active_ctas(total, p.ctas);
  if (static_cast<long long>(blockIdx.x) >= active) return;
  const long long begin = range_begin(blockIdx.x, total, active);
  const long long end = range_begin(blockIdx.x + 1, total, active);
  const int page = p.c.page;
  const int box = min(page, kTile);  // tokens per load

  if (warp == kConsumers) {
    // -------------------------------------------------------------- fetch
    int seq = 0;
    bool ok = true;
    for (long long u = begin; ok && u < end;) {
      const Segment g = segment_at(s_base, p.c.batch, pairs, u, end);
      const int head = g.pair / p.row_tiles;
      const int used = (kv_length(p.c, g.b, status) + page - 1) / page;  // pages that hold tokens
      int batch0 = -32;  // first of the 32 pages whose numbers and scales the lanes hold
      int id = -1;
      float kf = 0.f, ev = 0.f;
      for (int j = g.tile0; j < g.tile0 + g.tiles; ++j, ++seq) {
        const int first = j * kTile / page;
        if (first >= batch0 + 32 || batch0 < 0) {
          batch0 = first;
          const int at = batch0 + lane;
          id = at < used ? p.c.table[g.b * p.c.table_ld + at] : -1;
          if (at < used && (id < 0 || id >= p.c.pages)) {
            set_bad_shape(status);
            id = -1;
          }
          kf = 0.f;
          ev = 0.f;
          if (id >= 0) {
            const long long unit = static_cast<long long>(id) * p.c.kv_heads + head;
            kf = fp8_pow2(p.c.k_scale[unit] - 127) * p.scale_log2;
            ev = static_cast<float>(p.c.v_scale[unit] - 127);
          }
        }
        const int st = seq % C::kStages;
        const int loads = kTile / box;  // pages of this tile (1 where a page holds two tiles)
        const int mine = first + lane - batch0;
        const int my_id = __shfl_sync(0xffffffffu, id, mine & 31);
        const float my_kf = __shfl_sync(0xffffffffu, kf, mine & 31);
        const float my_ev = __shfl_sync(0xffffffffu, ev, mine & 31);
        ok = warp_wait(&empty[st], (static_cast<uint32_t>(seq / C::kStages) & 1u) ^ 1u, abort_flag, status);
        if (!ok) break;
        const bool load = lane < loads && my_id >= 0;
        if (lane < loads) s_meta[st * 4 + lane] = make_float2(my_kf, my_ev);
        const int count = __popc(__ballot_sync(0xffffffffu, load));
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(count) * 2 * box * D);
        __syncwarp();
        if (load) {
          // rows of the (pages x heads x tokens, D) code matrix
          const int row = (my_id * p.c.kv_heads + head) * page + (j * kTile) % page;
          uint8_t* dst = smem + st * C::kStageBytes + lane * box * D;
          tma_load_2d(dst, &kmap, &full[st], 0, row);
          tma_load_2d(dst + C::kTileBytes, &vmap, &full[st], 0, row);
        }
      }
      u += g.tiles;
    }
    if (*abort_flag) {
      volatile int never = 0;
      for (int back = 1; back <= min(seq, C::kStages); ++back)
        mbar_wait(&full[(seq - back) % C::kStages], static_cast<uint32_t>((seq - back) / C::kStages) & 1u, &never, status);
    }
  } else {
    // ------------------------------------------------------------ attend
    // Lane (g, c): rows g and g + 8, key g of a group of eight, channels
    // [c D/4, (c + 1) D/4) in q k; tokens 2c, 2c + 1, 2c + 8, 2c + 9 and
    // channels [g D/8, (g + 1) D/8) in p v.
    const int g = lane >> 2, c = lane & 3;
    constexpr int kSteps = D / 16;  // products over the channels
    constexpr int kCols = D / 8;    // groups of eight output columns
    int seq = 0;
    bool ok = true;
    for (long long u = begin; u < end;) {
      const Segment sg = segment_at(s_base, p.c.batch, pairs, u, end);
      const int head = sg.pair / p.row_tiles, row0 = (sg.pair % p.row_tiles) * kRows;
      const int len = kv_length(p.c, sg.b, status);
      // Queries as f16 fragments, their rows' power-of-two factors, and the keys a row sees.
      uint32_t qf[kSteps][4];
      float qs[2];
      int limit[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + g + 8 * h;
        const bool live = r < p.rows;
        const int i = live ? r / p.group : 0;
        limit[h] = !live ? len : (p.causal ? min(len, len - p.queries + i + 1) : len);
        float x[D / 4];
        if (live) {
          const T* src = static_cast<const T*>(p.q) + sg.b * p.q_batch + i * p.q_ld +
                         (static_cast<long long>(head) * p.group + r % p.group) * D + c * (D / 4);
          if (p.q_vec) {
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
              float t[8];
              load8<T>(src + 8 * k, t);
#pragma unroll
              for (int e = 0; e < 8; ++e) x[8 * k + e] = t[e];
            }
          } else {
#pragma unroll
            for (int k = 0; k < D / 4; ++k) x[k] = to_f32<T>(src[k]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < D / 4; ++k) x[k] = 0.f;
        }
        qs[h] = 1.f;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          // bf16 reaches past f16's range: bring the row's maximum to [1, 2)
          float m = 0.f;
#pragma unroll
          for (int k = 0; k < D / 4; ++k) m = fmaxf(m, fabsf(x[k]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const int e = min(126, max(-126, static_cast<int>(__float_as_uint(m) >> 23) - 127));
          qs[h] = fp8_pow2(e);
          const float inv = fp8_pow2(-e);
#pragma unroll
          for (int k = 0; k < D / 4; ++k) x[k] *= inv;
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          qf[s][h] = pack_half2(x[4 * s], x[4 * s + 1]);
          qf[s][2 + h] = pack_half2(x[4 * s + 2], x[4 * s + 3]);
        }
      }
      const int open = p.causal ? min(len, len - p.queries + row0 / p.group + 1) : len;  // keys that every row sees

      float o[kCols][4];
#pragma unroll
      for (int j = 0; j < kCols; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
      float top[2] = {kFloor, kFloor}, sum[2] = {0.f, 0.f};

      for (int t = 0; t < sg.tiles; ++t, ++seq) {
        if ((seq & (kConsumers - 1)) != warp) continue;
        const int st = seq % C::kStages;
        if (ok) ok = warp_wait(&full[st], static_cast<uint32_t>(seq / C::kStages) & 1u, abort_flag, status);
        if (!ok) continue;
        const uint8_t* sk = smem + st * C::kStageBytes;
        const uint8_t* sv = sk + C::kTileBytes;
        const int j0 = (sg.tile0 + t) * kTile;
        const bool masked = j0 + kTile > open;

        // Scores of 8 keys at a time.
        float s[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
          constexpr int W = D / 4 >= 16 ? 16 : D / 4;
          uint32_t w[D / 16];
#pragma unroll
          for (int h = 0; h < (D / 4) / W; ++h) {
            uint32_t part[W / 4];
            lds_words<W>(sk + swizzle_offset((8 * n + g) * D + c * (D / 4) + h * W, D), part);
#pragma unroll
            for (int e = 0; e < W / 4; ++e) w[h * (W / 4) + e] = part[e];
          }
#pragma unroll
          for (int k = 0; k < kSteps; ++k) mma16816(s[n], qf[k], fp8_unpack2(w[k] & 0xFFFFu), fp8_unpack2(w[k] >> 16));
        }
        uint32_t bad_lo = 0, bad_hi = 0;  // tokens some rows must not see whose values hold a NaN
        if (masked && p.queries > 1) {
          uint32_t any[2] = {0, 0};
#pragma unroll
          for (int h = 0; h < 2; ++h)
            for (int e = 0; e < D / 4; ++e)
              any[h] |= nan_codes(reinterpret_cast<const uint32_t*>(sv + (lane + 32 * h) * D)[e]);
          bad_lo = __ballot_sync(0xffffffffu, any[0] != 0);
          bad_hi = __ballot_sync(0xffffffffu, any[1] != 0);
        }
        float mx[2] = {kFloor, kFloor};
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 meta = s_meta[st * 4 + 8 * n / box];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = e >> 1;
            s[n][e] = fmaf(s[n][e], qs[h] * meta.x, meta.y);
            if (masked) {
              const int tok = 8 * n + 2 * c + (e & 1);
              if (((tok < 32 ? bad_lo >> tok : bad_hi >> (tok - 32)) & 1u) != 0) s[n][e] = fp8_nan();
              if (j0 + tok >= limit[h]) s[n][e] = -INFINITY;
            }
            mx[h] = fmaxf(mx[h], s[n][e]);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        }
        if (__any_sync(0xffffffffu, mx[0] > top[0] || mx[1] > top[1])) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float m = fmaxf(top[h], mx[h]);
            const float f = ex2_approx(top[h] - m);
            top[h] = m;
            sum[h] *= f;
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
              o[j][2 * h] *= f;
              o[j][2 * h + 1] *= f;
            }
          }
        }
        // Weights 2^(s + ev - M), packed as the A fragments of p v.
        uint32_t pf[8][2];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float undo = fp8_pow2(-static_cast<int>(s_meta[st * 4 + 8 * n / box].y));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float a = ex2_approx(s[n][2 * h] - top[h]), b = ex2_approx(s[n][2 * h + 1] - top[h]);
            sum[h] = fmaf(a + b, undo, sum[h]);
            pf[n][h] = pack_half2(a, b);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          constexpr int W = D / 8;
          uint32_t w[4][W / 4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = 16 * k + 2 * c + (e & 1) + 8 * (e >> 1);
            lds_words<W>(sv + swizzle_offset(tok * D + g * W, D), w[e]);
            if (masked) {
              const bool drop = j0 + tok >= len || (((tok < 32 ? bad_lo >> tok : bad_hi >> (tok - 32)) & 1u) != 0);
#pragma unroll
              for (int x = 0; x < W / 4; ++x)
                if (drop) w[e][x] = 0;
            }
          }
          const uint32_t a[4] = {pf[2 * k][0], pf[2 * k][1], pf[2 * k + 1][0], pf[2 * k + 1][1]};
#pragma unroll
          for (int x = 0; x < W / 4; ++x) {
            // channels 4x .. 4x + 3 of tokens (2c, 2c + 1) and (2c + 8, 2c + 9), paired by channel
            const uint32_t b0 = __byte_perm(w[0][x], w[1][x], 0x5140), b1 = __byte_perm(w[0][x], w[1][x], 0x7362);
            const uint32_t c0 = __byte_perm(w[2][x], w[3][x], 0x5140), c1 = __byte_perm(w[2][x], w[3][x], 0x7362);
            mma16816(o[4 * x], a, fp8_unpack2(b0 & 0xFFFFu), fp8_unpack2(c0 & 0xFFFFu));
            mma16816(o[4 * x + 1], a, fp8_unpack2(b0 >> 16), fp8_unpack2(c0 >> 16));
            mma16816(o[4 * x + 2], a, fp8_unpack2(b1 & 0xFFFFu), fp8_unpack2(c1 & 0xFFFFu));
            mma16816(o[4 * x + 3], a, fp8_unpack2(b1 >> 16), fp8_unpack2(c1 >> 16));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }

      // Merge the four warps.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        if (c == 0) {
          s_ml[(warp * kRows + g + 8 * h) * 2] = top[h];
          s_ml[(warp * kRows + g + 8 * h) * 2 + 1] = sum[h];
        }
      }
      named_barrier(1, kConsumers * 32);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        float m = kFloor;
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) m = fmaxf(m, s_ml[(w * kRows + r) * 2]);
        const float f = ex2_approx(top[h] - m);
        // column n = 2c + e of group j is channel n D/8 + j
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < kCols; ++j) s_o[(warp * kRows + r) * D + (2 * c + e) * kCols + j] = o[j][2 * h + e] * f;
      }
      named_barrier(1, kConsumers * 32);
      const int slot = blockIdx.x * 2 + (sg.tile0 == 0 ? 1 : 0);
      for (int at = threadIdx.x; at < kRows * D; at += kConsumers * 32) {
        const int r = at / D, d = at % D;
        if (row0 + r >= p.rows) continue;
        float m = kFloor, l = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) m = fmaxf(m, s_ml[(w * kRows + r) * 2]);
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) {
          l = fmaf(s_ml[(w * kRows + r) * 2 + 1], ex2_approx(s_ml[(w * kRows + r) * 2] - m), l);
          v += s_o[(w * kRows + r) * D + d];
        }
        if (sg.whole) {
          const int i = (row0 + r) / p.group;
          static_cast<T*>(p.out)[sg.b * p.out_batch + i * p.out_ld +
                                 (static_cast<long long>(head) * p.group + (row0 + r) % p.group) * D + d] =
              from_f32<T>(l == 0.f ? 0.f : v / l);
        } else {
          p.o_part[(static_cast<long long>(slot) * kRows + r) * D + d] = v;
          if (d == 0) {
            p.ml_part[(slot * kRows + r) * 2] = m;
            p.ml_part[(slot * kRows + r) * 2 + 1] = l;
          }
        }
      }
      named_barrier(1, kConsumers * 32);
      u += sg.tiles;
    }
  }
}

// One row of one (item, head, row tile): the partial results in the order of
// their tiles; zeros for an item without tokens.
template <int D, typename T>
__global__ void __launch_bounds__(128) kv_attention_merge_kernel(const AttnParams p, unsigned int* status) {
  __shared__ long long s_sum[2][4];
  pdl_begin();
  const int pairs = p.c.kv_heads * p.row_tiles;
  const int b = blockIdx.x / pairs, pair = blockIdx.x % pairs;
  long long total = 0, before = 0;
  for (int i = threadIdx.x; i < p.c.batch; i += 128) {
    const long long n = static_cast<long long>(tiles_of(kv_length(p.c, i, status))) * pairs;
    total += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane_id() == 0) {
    s_sum[0][warp_id()] = total;
    s_sum[1][warp_id()] = before;
  }
  __syncthreads();
  total = s_sum[0][0] + s_sum[0][1] + s_sum[0][2] + s_sum[0][3];
  before = s_sum[1][0] + s_sum[1][1] + s_sum[1][2] + s_sum[1][3];
  const int tiles = tiles_of(kv_length(p.c, b, status));
  const int head = pair / p.row_tiles, r = blockIdx.y, row = (pair % p.row_tiles) * kRows + r;
  if (row >= p.rows || static_cast<int>(threadIdx.x) >= D) return;
  T* out = static_cast<T*>(p.out) + b * p.out_batch + (row / p.group) * p.out_ld +
           (static_cast<long long>(head) * p.group + row % p.group) * D + threadIdx.x;
  if (tiles == 0) {
    *out = from_f32<T>(0.f);
    return;
  }
  const long long active = active_ctas(total, p.ctas);
  const long long u0 = before + static_cast<long long>(pair) * tiles, u1 = u0 + tiles;
  long long first = u0 * active / total;  // the CTA whose range holds u0
  while (range_begin(first + 1, total, active) <= u0) ++first;
  while (range_begin(first, total, active) > u0) --first;
  if (range_begin(first + 1, total, active) >= u1) return;  // one CTA had it all and wrote it
  float m = kFloor;
  for (long long cta = first; cta < active && range_begin(cta, total, active) < u1; ++cta) {
    const long long slot = cta * 2 + (range_begin(cta, total, active) <= u0 ? 1 : 0);
    m = fmaxf(m, p.ml_part[(slot * kRows + r) * 2]);
  }
  float l = 0.f, v = 0.f;
  for (long long cta = first; cta < active && range_begin(cta, total, active) < u1; ++cta) {
    const long long slot = cta * 2 + (range_begin(cta, total, active) <= u0 ? 1 : 0);
    const float f = ex2_approx(p.ml_part[(slot * kRows + r) * 2] - m);
    l = fmaf(p.ml_part[(slot * kRows + r) * 2 + 1], f, l);
    v = fmaf(p.o_part[(slot * kRows + r) * D + threadIdx.x], f, v);
  }
  *out = from_f32<T>(l == 0.f ? 0.f : v / l);
}

size_t partial_floats(int ctas, int head_dim) { return static_cast<size_t>(ctas) * 2 * kRows * (head_dim + 2); }

template <int D, typename T>
int launch(cudaStream_t stream, const CUtensorMap& kmap, const CUtensorMap& vmap, const AttnParams& p,
           unsigned int* status) {
  static unsigned long long configured = 0;
  const int most = 1024 + Cfg<D>::kOffBase + (kMaxBatch + 1) * 8;
  int rc = ensure_smem_attribute(reinterpret_cast<const void*>(kv_attention_kernel<D, T>), most, &configured,
                                 "kv_attention shared memory");
  if (rc != LDB_OK) return rc;
  const int smem = 1024 + Cfg<D>::kOffBase + (p.c.batch + 1) * 8;
  rc = launch_kernel(kv_attention_kernel<D, T>, dim3(p.ctas), dim3(kAttnThreads), smem, stream, "kv_attention launch",
                     kmap, vmap, p, status);
  if (rc != LDB_OK) return rc;
  const int pairs = p.c.batch * p.c.kv_heads * p.row_tiles;
  return launch_kernel(kv_attention_merge_kernel<D, T>, dim3(pairs, std::min(kRows, p.rows)), dim3(128), 0, stream,
                       "kv_attention merge launch", p, status);
}

template <typename T>
int launch_dim(cudaStream_t stream, const CUtensorMap& kmap, const CUtensorMap& vmap, const AttnParams& p, int head_dim,
               unsigned int* status) {
  if (head_dim == 32) return launch<32, T>(stream, kmap, vmap, p, status);
  if (head_dim == 64) return launch<64, T>(stream, kmap, vmap, p, status);
  return launch<128, T>(stream, kmap, vmap, p, status);
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_kv_attention_fp8_workspace_size(int batch, int queries, int heads, int kv_heads, int head_dim, size_t* bytes) {
  using namespace ldb;
  if (!bytes) return fail(LDB_ERR_INVALID, "kv_attention: bytes is null");
  if (batch < 0 || queries < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads ||
      (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return fail(LDB_ERR_SHAPE, "kv_attention: %d heads over %d of width %d (32, 64 or 128)", heads, kv_heads, head_dim);
  *bytes = partial_floats(kCtasPerSm * sm_count(), head_dim) * sizeof(float);
  return LDB_OK;
}

int ldb_kv_attention_fp8(cudaStream_t stream, const void* q, long long q_ld, long long q_batch, int dtype,
                         const uint8_t* k_codes, const uint8_t* v_codes, const uint8_t* k_scales,
                         const uint8_t* v_scales, int pages, int kv_heads, int page, int head_dim, const int* table,
                         long long table_ld, int width, const int* lengths, void* out, long long out_ld,
                         long long out_batch, int batch, int queries, int heads, float scale, int causal,
                         void* workspace, size_t workspace_bytes) {
  using namespace ldb;
  if (dtype != LDB_F16 && dtype != LDB_BF16) return fail(LDB_ERR_INVALID, "kv_attention: queries must be f16 or bf16");
  size_t need = 0;
  int rc = ldb_kv_attention_fp8_workspace_size(batch, queries, heads, kv_heads, head_dim, &need);
  if (rc != LDB_OK) return rc;
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return fail(LDB_ERR_SHAPE, "kv_attention: pages of %d tokens (16, 32, 64 or 128)", page);
  if (pages <= 0 || width <= 0 || table_ld < width || static_cast<long long>(width) * page > 0x7FFFFFFFll)
    return fail(LDB_ERR_SHAPE, "kv_attention: %d pages, table of %d", pages, width);
  const long long rows_all = static_cast<long long>(pages) * kv_heads * page;
  if (rows_all > 0x7FFFFFFFll) return fail(LDB_ERR_SHAPE, "kv_attention: cache of %lld token rows (2^31 - 1)", rows_all);
  if (batch > kMaxBatch) return fail(LDB_ERR_SHAPE, "kv_attention: at most %d items, got %d", kMaxBatch, batch);
  if (batch == 0 || queries == 0) return LDB_OK;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !table || !lengths || !out)
    return fail(LDB_ERR_INVALID, "kv_attention: null pointer");
  const long long row = static_cast<long long>(heads) * head_dim;
  if (queries > 1 && (q_ld < row || out_ld < row))
    return fail(LDB_ERR_SHAPE, "kv_attention: a row stride is below %lld", row);
  if (reinterpret_cast<uintptr_t>(k_codes) % 16 || reinterpret_cast<uintptr_t>(v_codes) % 16)
    return fail(LDB_ERR_ALIGNMENT, "kv_attention: codes must be 16-byte aligned");
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(LDB_ERR_WORKSPACE, "kv_attention needs %zu workspace bytes (16-byte aligned), got %zu", need,
                workspace_bytes);
  unsigned int* status = device_status_ptr();
  if (!status) return fail(LDB_ERR_CUDA, "kv_attention: no device status word");
  AttnParams p{};
  p.c = KvView{k_codes, v_codes, k_scales, v_scales, table, lengths, table_ld, pages, kv_heads, page, width, batch};
  p.q = q, p.q_ld = q_ld, p.q_batch = q_batch;
  p.out = out, p.out_ld = out_ld, p.out_batch = out_batch;
  p.queries = queries, p.group = heads / kv_heads;
  const long long group_rows = static_cast<long long>(queries) * p.group;
  const long long row_tiles = (group_rows + kRows - 1) / kRows;
  if (group_rows > 0x7FFFFFFFll || row_tiles * kv_heads * batch > 0x7FFFFFFFll)
    return fail(LDB_ERR_SHAPE, "kv_attention: too many query rows");
  p.rows = static_cast<int>(group_rows), p.row_tiles = static_cast<int>(row_tiles);
  p.causal = causal != 0;
  p.q_vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_ld % 8 == 0 && q_batch % 8 == 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.ctas = kCtasPerSm * sm_count();
  p.o_part = static_cast<float*>(workspace);
  p.ml_part = p.o_part + static_cast<size_t>(p.ctas) * 2 * kRows * head_dim;
  CUtensorMap kmap, vmap;
  const uint64_t dims[2] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(rows_all)};
  const uint64_t strides[1] = {static_cast<uint64_t>(head_dim)};
  const uint32_t box[2] = {static_cast<uint32_t>(head_dim), static_cast<uint32_t>(std::min(page, kTile))};
  rc = encode_tiled_u8(&kmap, k_codes, 2, dims, strides, box, head_dim);
  if (rc == LDB_OK) rc = encode_tiled_u8(&vmap, v_codes, 2, dims, strides, box, head_dim);
  if (rc != LDB_OK) return rc;
  return dtype == LDB_F16 ? launch_dim<__half>(stream, kmap, vmap, p, head_dim, status)
                          : launch_dim<__nv_bfloat16>(stream, kmap, vmap, p, head_dim, status);
}

}  // extern "C"
