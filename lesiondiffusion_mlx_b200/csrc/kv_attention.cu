// Attention of a few query rows over the paged 8-bit key/value cache.
//
//   s[r, j] = (q_r . k_j) 2^ek scale        over the codes of key j's page
//   o_r = sum_j 2^(s - M) 2^ev v_j / sum_j 2^(s - M)     (s in log2 units)
//
// with one running reference per row, M = max_j (s[r, j] + ev_j), so that every
// weight 2^(s + ev - M + 15) of the value product lies in [0, 2^15] whatever the
// pages' scales are, and is rounded to f16 once; the sum takes the same weight
// times 2^-(ev + 15) in FP32.  (The 2^15 is f16's range above 1: a weight is rounded
// to its 11 bits down to 2^-29 of the largest and is lost below 2^-40.  Without it
// these were 2^-14 and 2^-25, and a key that takes 0.9998 of the weight, or a page of
// zero values beside pages of scale 2^-20, cost the rest of the output its bits.)
//
// q k runs on the codes as they are (m16n8k32 e4m3): a query row is scaled by a
// power of two and written as e4m3 parts, q = q0 + q1 / 16 + q2 / 256, two for
// bf16 (8 significant bits), three for f16 (11), exactly but for channels
// 2^-14 below the row's largest.  The first two parts of eight rows fill the 16 rows
// of one product.  p v takes the values as f16 (exact) in the other
// orientation, channels x rows, so that eight rows fill the eight columns of
// a product and the scores' registers are its weight fragment as they are.
//
// Bound: HBM, the cached tokens (2 D bytes each) read once for a group's
// heads.  The cached tokens of all items and heads form one line of 32-token
// tiles, cut into equal ranges, one per warp, so that ragged lengths and
// preallocated tables leave no SM idle.  A warp works by itself: it copies the
// next tiles into its own ring (cp.async, swizzled) while it works on one, and
// keeps M, sum and output in registers until a pair of item and head ends, so
// that nothing waits for another warp.  A pair whose tiles lie in several
// ranges is merged by a second kernel, in order.  A lane's 16-byte reads of a
// swizzled row are free of bank conflicts, and the orders of channels (in q k)
// and of output rows (in p v) are chosen so that these bytes are its fragments.
//
// One B200, 8 heads of 128 shared by 4 bf16 queries each: 131072 tokens 53.4
// us (50 in this kernel, 5.4 TB/s; the start and the merge are the rest), 48 items
// of up to 8192 tokens 74 us (5.4 TB/s).  Tiles fetched by one warp per CTA
// with TMA and shared by four others took 74 and 154 us: the fetch was bound by
// the issue of its loads, and every change of pair by the four warps' barriers.

#include <algorithm>

#include "host_common.h"
#include "kv_attention.cuh"
#include "kv_attention_ranges.cuh"

namespace ldb {
namespace {

constexpr int kTile = 32;        // tokens per tile
constexpr int kGroupRows = 8;    // query rows of one product
// Positions on the line that the start of a pair counts for: its page numbers,
// scales and queries take a warp about as long as this many tiles.  (Without them a
// batch of 384 items of 2 to 1024 tokens took 166 us instead of 86.)
constexpr int kStart = 3;

// G groups of eight query rows per row tile.
template <int D, int G>
struct Cfg {
  static constexpr int kRows = G * kGroupRows;
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kSlotBytes = 2 * kTileBytes;
  // Tiles in flight: 16 KB a warp over eight to sixteen warps per SM, about
  // three times what HBM's latency times its rate asks for.
  static constexpr int kSlots = D == 128 ? 3 : (D == 64 ? 4 : 6);
  static constexpr int kCtasPerSm = D == 128 ? 2 : 3;
  static constexpr int kOffMeta = kWarps * kSlots * kSlotBytes;  // [warp][slot][2] (key factor, value exponent)
  static constexpr int kOffBase = kOffMeta + kWarps * kSlots * 16;  // [batch + 1] int
};
int ctas_per_sm(int head_dim) { return head_dim == 128 ? Cfg<128, 1>::kCtasPerSm : Cfg<64, 1>::kCtasPerSm; }

// ------------------------------------------------------------------ fragments

// D (16 x 8) += A (16 x 32) B (32 x 8), e4m3.
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A run of tiles of one (item, head, row tile) pair, and the copies of its
// tiles into the warp's ring.
template <int D, int G>
struct Fetch {
  const KvView& c;
  int b, head, used;      // pages that hold the item's tokens
  int batch0;             // first of the 32 pages whose numbers and scales the lanes hold
  int id;
  float kf, ev;
  float scale_log2;
  unsigned int* status;

  __device__ __forceinline__ Fetch(const KvView& view, float scale, unsigned int* st)
      : c(view), scale_log2(scale), status(st) {}

  __device__ __forceinline__ void start(int item, int h, int len) {
    b = item;
    head = h;
    used = (len + c.page - 1) / c.page;
    batch0 = -32;
  }

  // Copy tile j into the slot at `dst` (shared address) and its pages' factors to `meta`.
  __device__ __forceinline__ void tile(int j, uint32_t dst, float2* meta) {
    const int lane = lane_id();
    const int shift = 31 - __clz(c.page);
    const int first = (j * kTile) >> shift;
    if (first - batch0 > (c.page < kTile ? 30 : 31)) {
      batch0 = first;
      const int at = batch0 + lane;
      id = at < used ? c.table[b * c.table_ld + at] : -1;
      if (at < used && (id < 0 || id >= c.pages)) {
        set_bad_shape(status);
        id = -1;
      }
      kf = 0.f;
      ev = -INFINITY;  // (tokens of no page weigh nothing)
      if (id >= 0) {
        const long long unit = static_cast<long long>(id) * c.kv_heads + head;
        kf = fp8_pow2(c.k_scale[unit] - 127) * scale_log2;
        ev = static_cast<float>(c.v_scale[unit] - 127);
      }
    }
    const int at = first - batch0;
    const int id0 = __shfl_sync(0xffffffffu, id, at);
    const float kf0 = __shfl_sync(0xffffffffu, kf, at), ev0 = __shfl_sync(0xffffffffu, ev, at);
    int id1 = id0;
    float kf1 = kf0, ev1 = ev0;
    if (c.page < kTile) {
      id1 = __shfl_sync(0xffffffffu, id, at + 1);
      kf1 = __shfl_sync(0xffffffffu, kf, at + 1);
      ev1 = __shfl_sync(0xffffffffu, ev, at + 1);
    }
    if (lane < 2) meta[lane] = lane == 0 ? make_float2(kf0, ev0) : make_float2(kf1, ev1);
    // 16-byte unit q of a tile goes to its swizzled place: within 512 bytes the
    // pattern depends on the lane, and for 128-byte rows on the parity of i.
    constexpr int kUnits = kTile * D / 16 / 32;  // per lane, of K and of V
    const uint32_t even = swizzle_offset(lane * 16, D), odd = swizzle_offset(512 + lane * 16, D) - 512;
    const int inside = (j * kTile) & (c.page - 1);  // first row of the tile in its page
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // rows 0 .. 15 and 16 .. 31
      const int page_id = h == 0 ? id0 : id1;
      const int row = c.page < kTile ? 0 : inside + 16 * h;
      const long long off =
          ((static_cast<long long>(max(page_id, 0)) * c.kv_heads + head) * c.page + row) * D + lane * 16;
      const uint32_t bytes = page_id < 0 ? 0u : 16u;  // zeros for what has no page
#pragma unroll
      for (int i = 0; i < kUnits / 2; ++i) {
        const int at_i = h * (kUnits / 2) + i;
        const uint32_t to = dst + at_i * 512 + ((at_i & 1) ? odd : even);
        cp_async16(to, c.k + off + i * 512, bytes);
        cp_async16(to + kTile * D, c.v + off + i * 512, bytes);
      }
    }
  }
};

template <int D, int G, typename T>
__global__ void __launch_bounds__(kWarps * 32, Cfg<D, G>::kCtasPerSm)
    kv_attention_kernel(const AttnParams p, unsigned int* status) {
  using C = Cfg<D, G>;
  constexpr bool kThreeParts = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t smem[];
  int* s_base = reinterpret_cast<int*>(smem + C::kOffBase);
  const int warp = warp_id(), lane = lane_id();
  const int me = blockIdx.x * kWarps + warp;
  pdl_begin();
  const int pairs = p.c.kv_heads * p.row_tiles;
  lay_out_line<kTile, kStart>(p.c, pairs, s_base, status);
  clear_idle<T, D>(p, s_base);
  const Ranges ranges(s_base[p.c.batch], p.warps);
  const int begin = ranges.begin(me), end = ranges.begin(me + 1);
  if (!p.open_by_pair && lane == 0) p.open_part[me] = make_int4(0, 0, 0, 0);
  if (begin == end) return;

  const uint32_t ring = smem_u32(smem + warp * C::kSlots * C::kSlotBytes);
  const uint8_t* ring_ptr = smem + warp * C::kSlots * C::kSlotBytes;
  float2* s_meta = reinterpret_cast<float2*>(smem + C::kOffMeta) + warp * C::kSlots * 2;

  // Lane (g, c) holds, in q k, query row g of each group, keys 2c and 2c + 1
  // of every eight, channels [c D/4, (c + 1) D/4) of key g; in p v, tokens 2c, 2c
  // + 1, 2c + 8, 2c + 9 of every 16 and channels [g D/8, (g + 1) D/8), and the
  // outputs of those channels for rows 2c and 2c + 1.
  const int g = lane >> 2, c = lane & 3;
  constexpr int kSteps = D / 32;  // q k products over the channels
  constexpr int kMTiles = D / 16; // p v products over the channels
  // Swizzled places of the lane's bytes: the rows 8 n + g of K and 16 k + 8 h
  // + 2c (+ 1) of V have the same pattern for every n, k and h.
  constexpr int kWk = D / 4 >= 16 ? 16 : D / 4;  // bytes per read of K
  constexpr int kWv = D / 8;                     // bytes per read of V
  uint32_t at_k[(D / 4) / kWk], at_v[2];
#pragma unroll
  for (int h = 0; h < (D / 4) / kWk; ++h) at_k[h] = swizzle_offset(g * D + c * (D / 4) + h * kWk, D);
#pragma unroll
  for (int e = 0; e < 2; ++e) at_v[e] = C::kTileBytes + swizzle_offset((2 * c + e) * D + g * kWv, D);

  // The item and pair where the range begins.
  int b = 0;
  for (int lo = 0, hi = p.c.batch; hi - lo > 1;) {
    const int mid = (lo + hi) / 2;
    if (s_base[mid] <= begin) {
      lo = mid;
    } else {
      hi = mid;
    }
    b = lo;
  }
  Fetch<D, G> fetch(p.c, p.scale_log2, status);
  int places = (s_base[b + 1] - s_base[b]) / pairs;
  int pair = (begin - s_base[b]) / places;
  int at = s_base[b] + pair * places;  // of the pair
  for (; at < end; at += places, ++pair) {
    if (pair == pairs) {
      pair = 0;
      do {
        ++b;
      } while (s_base[b + 1] == s_base[b]);  // (position `at` exists, so a later item has tokens)
      places = (s_base[b + 1] - s_base[b]) / pairs;
    }
    const int item_tiles = places - kStart;
    const int tile0 = max(0, begin - at - kStart), tiles = min(item_tiles, end - at - kStart) - tile0;
    if (tiles <= 0) continue;
    const int head = pair / p.row_tiles, row0 = (pair % p.row_tiles) * C::kRows;
    const int len = kv_length(p.c, b, status);
    // Queries as they are, on their way while the page numbers arrive.
    uint32_t raw[G][D / 8];
    int limit[G];  // the keys a row sees
#pragma unroll
    for (int r = 0; r < G; ++r) {
      const int row = row0 + 8 * r + g;
      const bool live = row < p.rows;
      const int i = live ? row / p.group : 0;
      limit[r] = !live ? len : (p.causal ? min(len, len - p.queries + i + 1) : len);
      const T* src = static_cast<const T*>(p.q) + b * p.q_batch + i * p.q_ld +
                     (static_cast<long long>(head) * p.group + (live ? row % p.group : 0)) * D + c * (D / 4);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        if (!live) {
          raw[r][4 * k] = raw[r][4 * k + 1] = raw[r][4 * k + 2] = raw[r][4 * k + 3] = 0;
        } else if (p.q_vec) {
          const uint4 t = reinterpret_cast<const uint4*>(src)[k];
          raw[r][4 * k] = t.x, raw[r][4 * k + 1] = t.y, raw[r][4 * k + 2] = t.z, raw[r][4 * k + 3] = t.w;
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(src) + 8 * k;
#pragma unroll
          for (int e = 0; e < 4; ++e) raw[r][4 * k + e] = h[2 * e] | static_cast<uint32_t>(h[2 * e + 1]) << 16;
        }
      }
    }
    fetch.start(b, head, len);
#pragma unroll
    for (int t = 0; t < C::kSlots - 1; ++t) {
      if (t < tiles) fetch.tile(tile0 + t, ring + t * C::kSlotBytes, s_meta + 2 * t);
      cp_async_commit();
    }

    // Queries in parts, and their rows' power-of-two factors.
    uint32_t q01[G][kSteps][4];                   // parts 0 and 1 of four + four channels
    uint32_t q2[G][kThreeParts ? kSteps : 1][2];  // part 2
    float qs[G];
#pragma unroll
    for (int r = 0; r < G; ++r) {
      // the row's largest magnitude to [128, 256); a NaN stays one, an infinity makes the row's factor one
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < D / 8; ++k) {
        const float2 x = kv_unpack2<T>(raw[r][k]);
        m = fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y)));
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const int e = kv_query_exponent(m);
      qs[r] = fp8_is_finite(m) ? fp8_pow2(e - 7) : fp8_nan();
      const float inv = fp8_pow2(7 - e);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 x = kv_unpack2<T>(raw[r][4 * s + 2 * h]), y = kv_unpack2<T>(raw[r][4 * s + 2 * h + 1]);
          __half2 t[2] = {__floats2half2_rn(x.x * inv, x.y * inv), __floats2half2_rn(y.x * inv, y.y * inv)};
          q01[r][s][2 * h] = kv_split_part<16>(t);
          q01[r][s][2 * h + 1] = kv_split_part<16>(t);
          if constexpr (kThreeParts) q2[r][s][h] = kv_split_part<16>(t);
        }
    }
    const int open = p.causal ? min(len, len - p.queries + row0 / p.group + 1) : len;  // keys that every row sees

    float o[G][kMTiles][4];
#pragma unroll
    for (int r = 0; r < G; ++r)
#pragma unroll
      for (int j = 0; j < kMTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][j][e] = 0.f;
    float top[G], sum[G];
#pragma unroll
    for (int r = 0; r < G; ++r) top[r] = kFloor, sum[r] = 0.f;
    float ev_top = -INFINITY;  // largest value exponent met

    int slot = 0;
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      // The slot of tile t - 1 is free: start tile t + kSlots - 1, then wait for tile t.
      {
        const int into = slot == 0 ? C::kSlots - 1 : slot - 1;
        if (t + C::kSlots - 1 < tiles)
          fetch.tile(tile0 + t + C::kSlots - 1, ring + into * C::kSlotBytes, s_meta + 2 * into);
        cp_async_commit();
      }
      cp_async_wait<C::kSlots - 1>();
      __syncwarp();
      const uint8_t* sk = ring_ptr + slot * C::kSlotBytes;
      const float2 meta[2] = {s_meta[2 * slot], s_meta[2 * slot + 1]};
      const int j0 = (tile0 + t) * kTile;
      const bool masked = j0 + kTile > open;

      // Scores plus the value scale's exponent, eight keys at a time.
      float s[G][4][2];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        uint32_t w[D / 16];
#pragma unroll
        for (int h = 0; h < (D / 4) / kWk; ++h) {
          uint32_t part[kWk / 4];
          lds_words<kWk>(sk + at_k[h] + n * 8 * D, part);
#pragma unroll
          for (int e = 0; e < kWk / 4; ++e) w[h * (kWk / 4) + e] = part[e];
        }
#pragma unroll
        for (int r = 0; r < G; ++r) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
            mma_e4m3(d, q01[r][k][0], q01[r][k][1], q01[r][k][2], q01[r][k][3], w[2 * k], w[2 * k + 1]);
          if constexpr (kThreeParts) {
            float d2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) mma_e4m3(d2, q2[r][k][0], 0u, q2[r][k][1], 0u, w[2 * k], w[2 * k + 1]);
            d[2] = fmaf(d2[0], 0.0625f, d[2]);
            d[3] = fmaf(d2[1], 0.0625f, d[3]);
          }
          const float f = qs[r] * meta[n >> 1].x;
          s[r][n][0] = fmaf(fmaf(d[2], 0.0625f, d[0]), f, meta[n >> 1].y);
          s[r][n][1] = fmaf(fmaf(d[3], 0.0625f, d[1]), f, meta[n >> 1].y);
        }
      }
      uint32_t bad = 0;  // tokens whose values hold a NaN, where some rows may not see them
      if (masked) {
        if (p.causal && p.queries > 1) {
          uint32_t any = 0;
          for (int e = 0; e < D / 4; ++e)
            any |= kv_nan_codes(reinterpret_cast<const uint32_t*>(sk + C::kTileBytes + lane * D)[e]);
          bad = __ballot_sync(0xffffffffu, any != 0 && j0 + lane < len);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tok = 8 * n + 2 * c + e;
#pragma unroll
            for (int r = 0; r < G; ++r)
              if (j0 + tok >= limit[r]) s[r][n][e] = -INFINITY;
          }
      }
      float mx[G];
      bool grew = false;
#pragma unroll
      for (int r = 0; r < G; ++r) {
        mx[r] = kFloor;
#pragma unroll
        for (int n = 0; n < 4; ++n) mx[r] = fmaxf(mx[r], fmaxf(s[r][n][0], s[r][n][1]));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        grew |= mx[r] > top[r];
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int r = 0; r < G; ++r) {
          const float m = fmaxf(top[r], mx[r]);
          const float half = ex2_approx(0.5f * (top[r] - m)), f = half * half;
          top[r] = m;
          sum[r] = kv_scaled(sum[r], half);
          const float f0 = __shfl_sync(0xffffffffu, f, 8 * c), f1 = __shfl_sync(0xffffffffu, f, 8 * c + 4);
#pragma unroll
          for (int j = 0; j < kMTiles; ++j) {
            o[r][j][0] *= f0;
            o[r][j][1] *= f1;
            o[r][j][2] *= f0;
            o[r][j][3] *= f1;
          }
        }
      }
      // Weights 2^(s + ev - M + kHeadroom): the fragments of p v as they are.
      ev_top = fmaxf(ev_top, fmaxf(meta[0].y, meta[1].y));
      const bool far[2] = {kv_far_below(meta[0].y, ev_top), kv_far_below(meta[1].y, ev_top)};
      uint32_t pf[G][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float undo =
            far[n >> 1] ? 0.f : fp8_pow2(-max(static_cast<int>(meta[n >> 1].y), -127) - kHeadroom);
#pragma unroll
        for (int r = 0; r < G; ++r) {
          const float ref = top[r] - kHeadroom;
          const float a = ex2_approx(s[r][n][0] - ref), bb = ex2_approx(s[r][n][1] - ref);
          sum[r] = fmaf(a + bb, undo, sum[r]);
          pf[r][n] = pack_half2(a, bb);
        }
      }
      if (far[0] || far[1]) {  // (rare)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int r = 0; r < G; ++r)
            if (far[n >> 1])
              sum[r] += ex2_approx(s[r][n][0] - meta[n >> 1].y - top[r]) + ex2_approx(s[r][n][1] - meta[n >> 1].y - top[r]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t w[4][kWv / 4];  // tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lds_words<kWv>(sk + at_v[e & 1] + (16 * k + 8 * (e >> 1)) * D, w[e]);
          if (masked) {
            const int tok = 16 * k + 2 * c + (e & 1) + 8 * (e >> 1);
#pragma unroll
            for (int x = 0; x < kWv / 4; ++x) {
              if (j0 + tok >= len) w[e][x] = 0;
              if ((bad >> tok) & 1u) w[e][x] = kv_without_nan(w[e][x]);
            }
          }
        }
#pragma unroll
        for (int x = 0; x < kWv / 4; ++x) {
          // channels 4x .. 4x + 3 of tokens (2c, 2c + 1) and (2c + 8, 2c + 9), paired by channel
          const uint32_t b0 = __byte_perm(w[0][x], w[1][x], 0x5140), b1 = __byte_perm(w[0][x], w[1][x], 0x7362);
          const uint32_t c0 = __byte_perm(w[2][x], w[3][x], 0x5140), c1 = __byte_perm(w[2][x], w[3][x], 0x7362);
          const uint32_t v0 = fp8_unpack2(b0 & 0xFFFFu), v1 = fp8_unpack2(b0 >> 16);
          const uint32_t v2 = fp8_unpack2(c0 & 0xFFFFu), v3 = fp8_unpack2(c0 >> 16);
          const uint32_t v4 = fp8_unpack2(b1 & 0xFFFFu), v5 = fp8_unpack2(b1 >> 16);
          const uint32_t v6 = fp8_unpack2(c1 & 0xFFFFu), v7 = fp8_unpack2(c1 >> 16);
#pragma unroll
          for (int r = 0; r < G; ++r) {
            mma_f16(o[r][2 * x], v0, v1, v2, v3, pf[r][2 * k], pf[r][2 * k + 1]);
            mma_f16(o[r][2 * x + 1], v4, v5, v6, v7, pf[r][2 * k], pf[r][2 * k + 1]);
          }
        }
      }
      // The NaN that the product left out, to the rows that see its token.
      for (uint32_t rest = bad; rest; rest &= rest - 1) {
        const int tok = __ffs(rest) - 1;
        uint32_t w[kWv / 4];
        lds_words<kWv>(sk + C::kTileBytes + swizzle_offset(tok * D + g * kWv, D), w);
#pragma unroll
        for (int r = 0; r < G; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool seen = j0 + tok < __shfl_sync(0xffffffffu, limit[r], 8 * c + 4 * e);
#pragma unroll
            for (int x = 0; x < D / 8; ++x)  // channel g D/8 + x
              if (seen && ((kv_nan_codes(w[x / 4]) >> (8 * (x % 4))) & 0x80u)) o[r][x / 2][2 * (x % 2) + e] = fp8_nan();
          }
      }
      __syncwarp();
      if (++slot == C::kSlots) slot = 0;
    }

    // The pair's rows, or this range's part of them.
    const bool whole = tiles == item_tiles;
    const int part = me * 2 + (tile0 == 0 ? 1 : 0);
#pragma unroll
    for (int r = 0; r < G; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      if (!whole && c == 0) {
        float* ml = p.ml_part + (static_cast<long long>(part) * C::kRows + 8 * r + g) * 2;
        ml[0] = top[r];
        ml[1] = sum[r];
      }
      const float l[2] = {__shfl_sync(0xffffffffu, sum[r], 8 * c), __shfl_sync(0xffffffffu, sum[r], 8 * c + 4)};
      // products j: rows g and g + 8 are channels g D/8 + 2j and + 1
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + 8 * r + 2 * c + e;
        if (row >= p.rows) continue;
        if (whole) {
          const float inv = l[e] == 0.f ? 0.f : fp8_pow2(-kHeadroom) / l[e];
          T* dst = static_cast<T*>(p.out) + b * p.out_batch + (row / p.group) * p.out_ld +
                   (static_cast<long long>(head) * p.group + row % p.group) * D + g * (D / 8);
          if (D >= 64 && p.out_vec) {
#pragma unroll
            for (int j = 0; j < kMTiles / 4; ++j) {
              const float v[8] = {o[r][4 * j][e] * inv,     o[r][4 * j][2 + e] * inv,     o[r][4 * j + 1][e] * inv,
                                  o[r][4 * j + 1][2 + e] * inv, o[r][4 * j + 2][e] * inv, o[r][4 * j + 2][2 + e] * inv,
                                  o[r][4 * j + 3][e] * inv, o[r][4 * j + 3][2 + e] * inv};
              store8<T>(dst + 8 * j, v);
            }
          } else {
#pragma unroll
            for (int j = 0; j < kMTiles; ++j) {
              dst[2 * j] = from_f32<T>(o[r][j][e] * inv);
              dst[2 * j + 1] = from_f32<T>(o[r][j][2 + e] * inv);
            }
          }
        } else {
          float* dst = p.o_part + (static_cast<long long>(part) * C::kRows + 8 * r + 2 * c + e) * D + g * (D / 8);
#pragma unroll
          for (int j = 0; j < kMTiles / 2; ++j)
            reinterpret_cast<float4*>(dst)[j] =
                make_float4(o[r][2 * j][e], o[r][2 * j][2 + e], o[r][2 * j + 1][e], o[r][2 * j + 1][2 + e]);
        }
      }
    }
    // The warp that starts a pair says who goes on with it.
    if (tile0 == 0 && lane == 0 && (p.open_by_pair || !whole))
      p.open_part[p.open_by_pair ? b * pairs + pair : me] =
          make_int4(b, pair, me, whole ? 0 : ranges.of(at + kStart + item_tiles - 1) - me + 1);
  }
}

// Groups of eight query rows that one pass over the cache serves: as few as
// hold the rows, so that a lane's output stays in registers (8 D / 32 a group).
int row_groups(long long rows) { return rows <= 8 ? 1 : 2; }

// Rows from which on the 128-row tiles of the many-row kernel are the faster in
// bf16.  16 items of up to 4096 tokens, 8 heads, us here and there: of 128 channels 49 and 74 for
// 32 rows, 65 and 74 for 48, 83 and 74 for 64; of 64 36 and 50, 48 and 51, 60 and 51; of 32 32 and
// 49, 43 and 49, 54 and 49.  32768 tokens of one item: of 128 43 and 48, 54 and 49, 66 and 49;
// of 32 25 and 35, 33 and 35, 47 and 36.  f16, with its third part of the queries and, at 128
// channels, spilled registers, is past that point at 48 rows (of 128 123 and 79, of 64 66 and 52, of
// 32 48 and 50); the workspace's size is asked for without the type, so that the rule has none.
constexpr long long kTileRows = 49;

template <int D, int G, typename T>
int launch(cudaStream_t stream, const AttnParams& p, unsigned int* status) {
  static unsigned long long configured = 0;
  int rc = ensure_smem_attribute(reinterpret_cast<const void*>(kv_attention_kernel<D, G, T>),
                                 Cfg<D, G>::kOffBase + (kMaxBatch + 1) * 4, &configured, "kv_attention shared memory");
  if (rc != LDB_OK) return rc;
  rc = launch_kernel(kv_attention_kernel<D, G, T>, dim3(p.warps / kWarps), dim3(kWarps * 32),
                     Cfg<D, G>::kOffBase + (p.c.batch + 1) * 4, stream, "kv_attention launch", p, status);
  if (rc != LDB_OK) return rc;
  return launch_merge<D, T>(stream, p, kTile);
}

template <int D, typename T>
int launch_groups(cudaStream_t stream, const AttnParams& p, unsigned int* status) {
  return p.tile_rows == 8 ? launch<D, 1, T>(stream, p, status) : launch<D, 2, T>(stream, p, status);
}

template <typename T>
int launch_dim(cudaStream_t stream, const AttnParams& p, int head_dim, unsigned int* status) {
  if (head_dim == 32) return launch_groups<32, T>(stream, p, status);
  if (head_dim == 64) return launch_groups<64, T>(stream, p, status);
  return launch_groups<128, T>(stream, p, status);
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_kv_attention_fp8_table_workspace_size(int batch, int queries, int heads, int kv_heads, int head_dim,
                                              long long capacity, size_t* bytes) {
  using namespace ldb;
  if (!bytes) return fail(LDB_ERR_INVALID, "kv_attention: bytes is null");
  if (batch < 0 || queries < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads ||
      (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return fail(LDB_ERR_SHAPE, "kv_attention: %d heads over %d of width %d (32, 64 or 128)", heads, kv_heads, head_dim);
  const long long rows = static_cast<long long>(queries) * (heads / kv_heads);
  *bytes = rows >= kTileRows ? kv_tile_workspace(batch, kv_heads, rows, head_dim, capacity)
                             : workspace_bytes_of(ctas_per_sm(head_dim) * sm_count() * kWarps,
                                                  kGroupRows * row_groups(rows), head_dim);
  return LDB_OK;
}

int ldb_kv_attention_fp8_workspace_size(int batch, int queries, int heads, int kv_heads, int head_dim, size_t* bytes) {
  return ldb_kv_attention_fp8_table_workspace_size(batch, queries, heads, kv_heads, head_dim, -1, bytes);
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
  int rc = ldb_kv_attention_fp8_table_workspace_size(batch, queries, heads, kv_heads, head_dim,
                                                     static_cast<long long>(std::max(width, 0)) * std::max(page, 0),
                                                     &need);
  if (rc != LDB_OK) return rc;
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return fail(LDB_ERR_SHAPE, "kv_attention: pages of %d tokens (16, 32, 64 or 128)", page);
  if (pages <= 0 || width <= 0 || table_ld < width || static_cast<long long>(width) * page > 0x7FFFFFFFll)
    return fail(LDB_ERR_SHAPE, "kv_attention: %d pages, table of %d", pages, width);
  const long long rows_all = static_cast<long long>(pages) * kv_heads * page;
  if (rows_all > 0x7FFFFFFFll)
    return fail(LDB_ERR_SHAPE, "kv_attention: cache of %lld token rows (2^31 - 1)", rows_all);
  if (batch > kMaxBatch) return fail(LDB_ERR_SHAPE, "kv_attention: at most %d items, got %d", kMaxBatch, batch);
  if (batch == 0 || queries == 0) return LDB_OK;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !table || !lengths || !out)
    return fail(LDB_ERR_INVALID, "kv_attention: null pointer");
  const long long row = static_cast<long long>(heads) * head_dim;
  if ((queries > 1 && (q_ld < row || out_ld < row)) || (batch > 1 && out_batch < row))
    return fail(LDB_ERR_SHAPE, "kv_attention: a row stride, or the output's item stride, is below %lld", row);
  if (reinterpret_cast<uintptr_t>(k_codes) % 16 || reinterpret_cast<uintptr_t>(v_codes) % 16)
    return fail(LDB_ERR_ALIGNMENT, "kv_attention: codes must be 16-byte aligned");
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(LDB_ERR_WORKSPACE, "kv_attention needs %zu workspace bytes (16-byte aligned), got %zu", need,
                workspace_bytes);
  unsigned int* status = device_status_ptr();
  if (!status) return fail(LDB_ERR_CUDA, "kv_attention: no device status word");
  const KvView view{k_codes,  v_codes, k_scales, v_scales, table, lengths,
                    table_ld, pages,   kv_heads, page,     width, batch};
  const long long group_rows = static_cast<long long>(queries) * (heads / kv_heads);
  if (group_rows > 0x7FFFFF00ll) return fail(LDB_ERR_SHAPE, "kv_attention: too many query rows");
  const int q_vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_ld % 8 == 0 && q_batch % 8 == 0;
  const int out_vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_ld % 8 == 0 && out_batch % 8 == 0;
  if (group_rows >= kTileRows) {
    KvTileParams t{};
    t.c = view;
    t.q = q, t.q_ld = q_ld, t.q_batch = q_batch, t.q_vec = q_vec;
    t.out = out, t.out_ld = out_ld, t.out_batch = out_batch, t.out_vec = out_vec;
    t.queries = queries, t.group = heads / kv_heads, t.rows = static_cast<int>(group_rows), t.causal = causal != 0;
    return kv_attention_tiles(stream, t, head_dim, dtype, scale, workspace, status);
  }
  AttnParams p{};
  p.c = view;
  p.q = q, p.q_ld = q_ld, p.q_batch = q_batch, p.q_vec = q_vec;
  p.out = out, p.out_ld = out_ld, p.out_batch = out_batch, p.out_vec = out_vec;
  p.queries = queries, p.group = heads / kv_heads;
  p.tile_rows = kGroupRows * row_groups(group_rows);
  const long long row_tiles = (group_rows + p.tile_rows - 1) / p.tile_rows;
  const long long tiles = kStart + (static_cast<long long>(width) * page + kTile - 1) / kTile;
  if (row_tiles * kv_heads > 0x7FFFFFFFll || row_tiles * kv_heads * batch * tiles > 0x7FFFFFFFll)
    return fail(LDB_ERR_SHAPE, "kv_attention: too many heads over too long a table");
  p.rows = static_cast<int>(group_rows), p.row_tiles = static_cast<int>(row_tiles);
  p.causal = causal != 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.warps = ctas_per_sm(head_dim) * sm_count() * kWarps;
  p.o_part = static_cast<float*>(workspace);
  p.ml_part = p.o_part + static_cast<size_t>(p.warps) * 2 * p.tile_rows * head_dim;
  p.open_by_pair = row_tiles * kv_heads * batch <= p.warps;
  p.status = status;
  p.open_part = reinterpret_cast<int4*>(p.ml_part + static_cast<size_t>(p.warps) * 2 * p.tile_rows * 2);
  return dtype == LDB_F16 ? launch_dim<__half>(stream, p, head_dim, status)
                          : launch_dim<__nv_bfloat16>(stream, p, head_dim, status);
}

}  // extern "C"
