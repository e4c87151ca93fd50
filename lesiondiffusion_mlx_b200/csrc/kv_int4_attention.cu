// Attention of a few query rows over the paged 4-bit key/value cache.
//
//   o_r = sum_j 2^(s[r, j] - M) v_j / sum_j 2^(s[r, j] - M),   s[r, j] = q_r . k_j scale log2(e)
//
// with a running reference M per row.  Codes become f16 on the way to the tensor
// cores (m16n8k16): a code in bits 4 .. 7 of an f16 whose upper bits are those of 64 is 64 +
// code, and one fused multiply-add, (64 + code) s - 72 s, is the value, exactly.  A
// word's eight codes take three shifts and four three-input ANDs for four pairs.  Keys
// come out as pairs of channels, so the queries are paired like them; values of two
// neighbouring tokens are paired by exchanging half words first, and their scales come
// as pairs too.  Queries are f16 as they are, or bf16 rows scaled by a power of
// two (exact down to 2^-31 of the row's largest).  M follows a row's maximum only once that is 2^4 above
// it, so that most tiles scale nothing.  Weights are rounded to f16 once, 2^11 at M (within f16 at 2^15), with
// 11 bits down to 2^-25 of M and lost below 2^-36; their sum is FP32.
//
// Bound: HBM, (D / 2 + D / 16) 2 bytes a token and key/value head, read once for
// a group's heads.  The tiles of 32 tokens of all items and heads form one line that the
// warps share out equally (kv_attention_ranges.cuh); a warp copies the next
// tiles into its own ring (cp.async) while it works on one.
//
// One B200, one bf16 token of 32 heads of 128 over 8: behind 262144 tokens 70 us (302 MB at
// 4.3 TB/s: 8 of them in the join of its warps' parts), behind 32 items of up to 16384 71 us.  Of
// the kernel's issue slots 62 % are taken, most by unpacking; without the unpacking it would be
// bound by HBM.

#include <algorithm>
#include <cmath>

#include "host_common.h"
#include "kv_attention.cuh"
#include "kv_attention_ranges.cuh"
#include "kv_int4.cuh"
#include "kv_int4_attention.cuh"

namespace ldb {
namespace {

constexpr int kTile = 32;      // tokens per tile
constexpr int kKeys = kTile / 8;      // q k products of a tile: eight keys each
constexpr int kLaneTokens = kTile / 4;
constexpr int kChunks = kTile / 16;   // of 16 tokens, each of one page
constexpr float kLag = 4.f;           // a reference follows its row's maximum once that is 2^4 above
constexpr int kHeadroomLag = kHeadroom - 4;
constexpr int kGroupRows = 8;  // query rows of one value product
// Positions on the line that the start of a pair counts for.
constexpr int kStart = 3;

// An 8 x 8 matrix of 16-bit values, a pair of a row's neighbours per lane, transposed.
__device__ __forceinline__ uint32_t transposed8(uint32_t w) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(w));
  return d;
}

// CTAs an SM, as far as registers allow.  One group, 262144 tokens of 128 channels, us: two 72, three 71, four (128 registers
// a thread) 76; of 64 channels 50 with four, 47 with three.
constexpr int ctas_of(int head_dim, int groups) { return groups == 1 ? 3 : (head_dim == 128 ? 2 : 3); }

// G groups of eight query rows per row tile.
template <int D, int G>
struct Cfg {
  static constexpr int kRows = G * kGroupRows;
  static constexpr int kTokenBytes = D / 2;
  static constexpr int kGroups = D / kInt4Group;
  static constexpr int kCodeBytes = kTile * kTokenBytes;
  static constexpr int kScaleBytes = kGroups * kTile;
  static constexpr int kOffScale = 2 * kCodeBytes;  // in a slot: codes of K and V, then scales of K and V
  static constexpr int kSlotBytes = 2 * (kCodeBytes + kScaleBytes);
  static constexpr int kSlots = D == 128 ? 3 : (D == 64 ? 6 : 8);
  static constexpr int kCtasPerSm = ctas_of(D, G);
  static constexpr int kOffBase = kWarps * kSlots * kSlotBytes;  // [batch + 1] int
};
// A run of tiles of one (item, head, row tile) pair, and the copies of its tiles into the warp's ring.
template <int D>
struct Fetch {
  using C = Cfg<D, 1>;
  const KvView& c;
  const int* pages;   // of the item
  int head, used;     // pages that hold the item's tokens
  int batch0;         // first of the 32 pages whose numbers the lanes hold
  int id, shift;
  bool lost;          // the table has named a page wrongly
  // The lane's: 16 bytes of codes in a run of 512, and its 16 tokens of a group's scales (of keys, then of values).
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* scale;
  int scale_to, group;  // (negative: none)
  unsigned int* status;

  __device__ __forceinline__ Fetch(const KvView& view, unsigned int* st) : c(view), status(st) {
    const int lane = lane_id();
    const int which = lane / (kChunks * C::kGroups);
    shift = 31 - __clz(view.page);
    group = (lane / kChunks) % C::kGroups;
    k = view.k + lane * 16;
    v = view.v + lane * 16;
    scale = which ? view.v_scale : view.k_scale;
    scale_to = which < 2 ? C::kOffScale + (which * C::kGroups + group) * kTile + lane % kChunks * 16 : -1;
  }

  __device__ __forceinline__ void start(int item, int h, int len) {
    pages = c.table + item * c.table_ld;
    head = h;
    used = (len + c.page - 1) >> shift;
    batch0 = -32;
    lost = false;
  }

  // Copy tile j into slot `slot` of the ring at `ring` (shared address).
  __device__ __forceinline__ void tile(int j, uint32_t ring, int slot) {
    const uint32_t dst = ring + slot * C::kSlotBytes;
    const int lane = lane_id();
    const int first = (j * kTile) >> shift;
    if (first - batch0 > 32 - kChunks) {  // (a tile has up to kChunks pages)
      batch0 = first;
      const int at = batch0 + lane;
      id = at < used ? pages[at] : -1;
      if (at < used && (id < 0 || id >= c.pages)) {
        set_bad_shape(status);
        id = -1;
      }
    }
    const int at = first - batch0;
    const uint32_t to = dst + lane * 16;
    const int page0 = __shfl_sync(0xffffffffu, id, at);
    lost |= page0 < 0;
    const uint32_t bytes0 = page0 < 0 ? 0u : 16u;  // zeros for what has no page
    const int unit0 = max(page0, 0) * c.kv_heads + head;  // (the cache has fewer than 2^31 rows)
    if (c.page >= kTile) {  // one run of tokens
      const int in = (j * kTile) & (c.page - 1);
      const long long off = static_cast<long long>(unit0 * c.page + in) * C::kTokenBytes;
#pragma unroll
      for (int i = 0; i < kTile * C::kTokenBytes / 512; ++i) {
        cp_async16(to + i * 512, k + off + i * 512, bytes0);
        cp_async16(to + C::kCodeBytes + i * 512, v + off + i * 512, bytes0);
      }
      if (scale_to >= 0)
        cp_async16(dst + scale_to,
                   scale + static_cast<long long>(unit0 * C::kGroups + group) * c.page + in + (lane & 1) * 16, bytes0);
    } else {  // two pages of 16
      const int page1 = __shfl_sync(0xffffffffu, id, at + 1);
      lost |= page1 < 0 && first + 1 < used;
      const uint32_t bytes1 = page1 < 0 ? 0u : 16u;
      const int unit1 = max(page1, 0) * c.kv_heads + head;
#pragma unroll
      for (int i = 0; i < kTile * C::kTokenBytes / 512; ++i) {
        const bool n = (i * 512 + lane * 16) / (16 * C::kTokenBytes);  // second page
        const long long off =
            static_cast<long long>(n ? unit1 : unit0) * 16 * C::kTokenBytes + i * 512 - (n ? 16 * C::kTokenBytes : 0);
        cp_async16(to + i * 512, k + off, n ? bytes1 : bytes0);
        cp_async16(to + C::kCodeBytes + i * 512, v + off, n ? bytes1 : bytes0);
      }
      if (scale_to >= 0) {
        const bool n = lane & 1;
        cp_async16(dst + scale_to, scale + static_cast<long long>((n ? unit1 : unit0) * C::kGroups + group) * 16,
                   n ? bytes1 : bytes0);
      }
    }
  }

  // Whether the table names the page of token `tok` wrongly (asked where `lost` says that it does so anywhere).
  __device__ __forceinline__ bool is_lost(int tok) const {
    if (tok >> shift >= used) return false;
    const int page = pages[tok >> shift];
    return page < 0 || page >= c.pages;
  }
};

template <int D, int G, typename T>
__global__ void __launch_bounds__(kWarps * 32, Cfg<D, G>::kCtasPerSm)
    kv_int4_attention_kernel(const AttnParams p, unsigned int* status) {
  using C = Cfg<D, G>;
  constexpr bool kScaled = !std::is_same<T, __half>::value;  // rows scaled by a power of two
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

  // Lane (g, c) holds, in q k, channels [c D/4, (c + 1) D/4) of query row g of each group and of key
  // g of each of kKeys blocks of eight (two blocks a product), and key g's scores for
  // rows 2c and 2c + 1; in p v, the weights of row g for keys 2c and 2c + 1 of each block (the scores
  // transposed), those tokens' channels [g D/8, (g + 1) D/8), and their outputs for rows 2c and 2c + 1.  Key j of
  // block n is token 8 (j / 2) + 2n + (j % 2, the other way round for odd j / 2): so a
  // lane's tokens in p v are eight neighbours, whose scales are one 8-byte read, and
  // lanes that read codes at a time meet in a bank at most twice.
  const int g = lane >> 2, c = lane & 3;
  constexpr int kSteps = D / 16;            // q k products over the channels
  constexpr int kMTiles = D / 16;           // p v products over the channels
  constexpr int kWk = D / 8;                // bytes of a key's channels: 16, 8 or 4
  constexpr int kWv = D / 16;               // bytes of a value's: 8, 4 or 2
  const int odd_k = (g & 1) ^ ((g >> 1) & 1), odd_v = c & 1;
  const int at_k = (kLaneTokens * (g >> 1) + odd_k) * C::kTokenBytes + c * kWk;
  const int at_v = C::kCodeBytes + kLaneTokens * c * C::kTokenBytes + g * kWv;
  const int at_ks = C::kOffScale + (c * (D / 4) / kInt4Group) * kTile + kLaneTokens * (g >> 1);
  const int at_vs = C::kOffScale + C::kScaleBytes + (g * (D / 8) / kInt4Group) * kTile + kLaneTokens * c;
  const uint32_t sel_k[2] = {scale_selector(odd_k, odd_k), scale_selector(odd_k + 2, odd_k + 2)};
  const uint32_t sel_v[2] = {scale_selector(odd_v, 1 - odd_v), scale_selector(2 + odd_v, 3 - odd_v)};

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
  Fetch<D> fetch(p.c, status);
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
    int limit[G][2];  // the keys that rows 2c and 2c + 1 see
    float factor[G][2];
#pragma unroll
    for (int r = 0; r < G; ++r) {
      const int row = row0 + 8 * r + g;
      const bool live = row < p.rows;
      const int i = live ? row / p.group : 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int of = row0 + 8 * r + 2 * c + e;
        limit[r][e] = of < p.rows && p.causal ? min(len, len - p.queries + of / p.group + 1) : len;
      }
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
      if (t < tiles) fetch.tile(tile0 + t, ring, t);
      cp_async_commit();
    }

    // Queries in the channel order of the unpacked keys, and their rows' factors.
    uint32_t qa[G][kSteps][2];
#pragma unroll
    for (int r = 0; r < G; ++r) {
      // a NaN stays one, an infinity makes the row's factor one (of a row that sees any key)
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < D / 8; ++k) {
        const float2 x = kv_unpack2<T>(raw[r][k]);
        m = fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y)));
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const int e = kv_query_exponent(m);
      const float own = (kScaled ? fp8_pow2(e - 7) * 0.0078125f : 1.f) * p.scale_log2;
      const float size = fmaxf(own, 1.2e-38f);  // (-inf times zero would be a NaN)
      const bool finite = fp8_is_finite(m);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f = __shfl_sync(0xffffffffu, finite ? size : -size, 8 * c + 4 * x);
        factor[r][x] = f > 0.f ? f : (limit[r][x] <= 0 ? -f : fp8_nan());
      }
      if constexpr (kScaled) {
        const float inv = fp8_pow2(7 - e);  // largest magnitude to [2^7, 2^8), and then to [2^14, 2^15)
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          const float2 x = kv_unpack2<T>(raw[r][k]);
          raw[r][k] = pack_half2(x.x * inv * 128.f, x.y * inv * 128.f);
        }
      }
#pragma unroll
      for (int w = 0; w < D / 8; ++w) raw[r][w] ^= p.negate ? 0x80008000u : 0u;
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {  // channels 8 w .. 8 w + 7 of the lane's: pairs (n, n + 4)
        qa[r][2 * w][0] = __byte_perm(raw[r][4 * w], raw[r][4 * w + 2], 0x5410);
        qa[r][2 * w][1] = __byte_perm(raw[r][4 * w], raw[r][4 * w + 2], 0x7632);
        qa[r][2 * w + 1][0] = __byte_perm(raw[r][4 * w + 1], raw[r][4 * w + 3], 0x5410);
        qa[r][2 * w + 1][1] = __byte_perm(raw[r][4 * w + 1], raw[r][4 * w + 3], 0x7632);
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
    float top[G][2], sum[G][2];
#pragma unroll
    for (int r = 0; r < G; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) top[r][e] = kUnseen, sum[r][e] = 0.f;
    // Where a reference is far: the references and factors, in whose place `top` and `factor` are zero and one.
    bool far = false;
    float far_top[G][2], far_factor[G][2];

    int slot = 0;
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      // The slot of tile t - 1 is free: start tile t + kSlots - 1, then wait for tile t.
      {
        const int into = slot == 0 ? C::kSlots - 1 : slot - 1;
        if (t + C::kSlots - 1 < tiles) fetch.tile(tile0 + t + C::kSlots - 1, ring, into);
        cp_async_commit();
      }
      cp_async_wait<C::kSlots - 1>();
      __syncwarp();
      const uint8_t* sk = ring_ptr + slot * C::kSlotBytes;
      const int j0 = (tile0 + t) * kTile;
      const bool masked = j0 + kTile > open || fetch.lost;

      // Scores, eight keys at a time.
      float s[G][kKeys][2];
      {
        constexpr int kKeyGroups = D == 128 ? 2 : 1;  // of the lane's channels
        uint32_t scales[kKeyGroups][2];
#pragma unroll
        for (int h = 0; h < kKeyGroups; ++h) lds_words<8>(sk + at_ks + h * kTile, scales[h]);
#pragma unroll
        for (int n = 0; n < kKeys; n += 2) {
          uint32_t w[2][kWk / 4];
          lds_words<kWk>(sk + at_k + 2 * n * C::kTokenBytes, w[0]);
          lds_words<kWk>(sk + at_k + 2 * (n + 1) * C::kTokenBytes, w[1]);
          float d[G][4];
#pragma unroll
          for (int r = 0; r < G; ++r) d[r][0] = d[r][1] = d[r][2] = d[r][3] = 0.f;
#pragma unroll
          for (int i = 0; i < kWk / 4; ++i) {
            uint32_t v[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t sc = scale_pair(scales[kKeyGroups == 2 ? i >> 1 : 0][n >> 1], sel_k[h]);
              unpack4(w[h][i], as_half2(sc), minus72(sc), v[h]);
            }
#pragma unroll
            for (int r = 0; r < G; ++r) {
              mma_f16(d[r], v[0][0], v[1][0], v[0][1], v[1][1], qa[r][2 * i][0], qa[r][2 * i][1]);
              mma_f16(d[r], v[0][2], v[1][2], v[0][3], v[1][3], qa[r][2 * i + 1][0], qa[r][2 * i + 1][1]);
            }
          }
#pragma unroll
          for (int r = 0; r < G; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s[r][n + h][0] = d[r][2 * h];
              s[r][n + h][1] = d[r][2 * h + 1];
            }
        }
      }
      uint32_t vs[2];  // scales of the values of the lane's tokens
      lds_words<8>(sk + at_vs, vs);
      uint32_t bad = 0;  // tokens whose values are NaN in the lane's group, where some rows may not see them
      if (masked) {
#pragma unroll
        for (int n = 0; n < kKeys; ++n) {
          const int tok = kLaneTokens * (g >> 1) + 2 * n + odd_k;
          const bool gone = fetch.lost && fetch.is_lost(j0 + tok);
#pragma unroll
          for (int r = 0; r < G; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (j0 + tok >= limit[r][e] || gone) s[r][n][e] = -INFINITY;
        }
        const int left = len - j0 - kLaneTokens * c;  // of the lane's tokens, those that exist
        uint32_t mine = 0;
#pragma unroll
        for (int k = 0; k < kLaneTokens / 4; ++k) {
          const int n = min(max(left - 4 * k, 0), 4);
          vs[k] = n == 4 ? vs[k] : vs[k] & ((1u << (8 * n)) - 1u);
          if (p.causal && p.queries > 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (((vs[k] >> (8 * j)) & 0xFFu) == kInt4NanScale) {
                vs[k] &= ~(0xFFu << (8 * j));
                mine |= 1u << (4 * k + j);
              }
            }
          }
        }
        bad = mine << (kLaneTokens * c);
        bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
        bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
      }
      float mx[G][2];  // the lane's keys
      bool grew = false;
#pragma unroll
      for (int r = 0; r < G; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m = fmaxf(fmaxf(s[r][0][e], s[r][1][e]), fmaxf(s[r][2][e], s[r][3][e]));
          mx[r][e] = __fmul_rn(m, factor[r][e]);
          grew |= mx[r][e] > top[r][e] + kLag;
        }
      if (__any_sync(0xffffffffu, grew) || far) {
        bool wide = false;  // (of a far reference)
#pragma unroll
        for (int r = 0; r < G; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float was = far ? far_top[r][e] : top[r][e];
            float m = fmaxf(was, far ? __fmul_rn(mx[r][e], far_factor[r][e]) : mx[r][e]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float half = ex2_approx(0.5f * (was - m)), f = half * half;
            wide |= is_far(m);
            top[r][e] = m;
            sum[r][e] = kv_scaled(sum[r][e], half);
#pragma unroll
            for (int j = 0; j < kMTiles; ++j) {
              o[r][j][e] *= f;
              o[r][j][2 + e] *= f;
            }
          }
        if (far || __any_sync(0xffffffffu, wide)) {
#pragma unroll
          for (int r = 0; r < G; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (!far) far_factor[r][e] = factor[r][e];
              far_top[r][e] = top[r][e], top[r][e] = 0.f, factor[r][e] = 1.f;
#pragma unroll
              for (int n = 0; n < kKeys; ++n) s[r][n][e] = __fmul_rn(s[r][n][e], far_factor[r][e]) - far_top[r][e];
            }
          far = true;
        }
      }
      // Weights 2^(s - M + kHeadroomLag), transposed: the fragments of p v.
      uint32_t pf[G][kKeys];
#pragma unroll
      for (int r = 0; r < G; ++r) {
        const float ref0 = kHeadroomLag - top[r][0], ref1 = kHeadroomLag - top[r][1];
#pragma unroll
        for (int n = 0; n < kKeys; ++n) {
          const float a = ex2_approx(fmaf(s[r][n][0], factor[r][0], ref0));
          const float bb = ex2_approx(fmaf(s[r][n][1], factor[r][1], ref1));
          sum[r][0] += a;
          sum[r][1] += bb;
          pf[r][n] = transposed8(pack_half2(a, bb));
        }
      }
#pragma unroll
      for (int k = 0; k < kLaneTokens / 4; ++k) {
        // tokens (columns 2c, 2c + 1) of products 2k and 2k + 1, their channels paired by token
        constexpr int kWords = (kWv + 3) / 4;
        uint32_t w[4][kWords];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint8_t* from = sk + at_v + (4 * k + 2 * (e >> 1) + ((e & 1) ^ odd_v)) * C::kTokenBytes;
          if constexpr (kWv == 2) {
            w[e][0] = *reinterpret_cast<const uint16_t*>(from);
          } else {
            lds_words<kWv>(from, w[e]);
          }
        }
        const uint32_t s0 = scale_pair(vs[k], sel_v[0]), s1 = scale_pair(vs[k], sel_v[1]);
        const __half2 m0 = minus72(s0), m1 = minus72(s1);
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {  // four channels 4x .. 4x + 3 of the lane's
          const uint32_t sel = x & 1 ? 0x7632 : 0x5410;
          uint32_t v0[4], v1[4];
          unpack4(__byte_perm(w[0][x >> 1], w[1][x >> 1], sel), as_half2(s0), m0, v0);
          unpack4(__byte_perm(w[2][x >> 1], w[3][x >> 1], sel), as_half2(s1), m1, v1);
#pragma unroll
          for (int r = 0; r < G; ++r) {
            mma_f16(o[r][2 * x], v0[0], v0[1], v1[0], v1[1], pf[r][2 * k], pf[r][2 * k + 1]);
            mma_f16(o[r][2 * x + 1], v0[2], v0[3], v1[2], v1[3], pf[r][2 * k], pf[r][2 * k + 1]);
          }
        }
      }
      if (__any_sync(0xffffffffu, bad != 0)) {
        // Rare: the NaN that the product left out, to the rows that see its token.
#pragma unroll
        for (int r = 0; r < G; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int seen = limit[r][e] - j0;  // of the tile's tokens
            const uint32_t in = seen <= 0 ? 0 : (seen >= kTile ? ~0u : (1u << seen) - 1);
            if (bad & in) {
#pragma unroll
              for (int j = 0; j < kMTiles; ++j) o[r][j][e] = o[r][j][2 + e] = fp8_nan();
            }
          }
      }
      __syncwarp();
      if (++slot == C::kSlots) slot = 0;
    }

    // The pair's rows, or this range's part of them.
    if (far) {
#pragma unroll
      for (int r = 0; r < G; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) top[r][e] = far_top[r][e];
    }
    const bool whole = tiles == item_tiles;
    const int part = me * 2 + (tile0 == 0 ? 1 : 0);
#pragma unroll
    for (int r = 0; r < G; ++r) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[r][e] += __shfl_xor_sync(0xffffffffu, sum[r][e], o);
        if (!whole && g == 0) {
          float* ml = p.ml_part + (static_cast<long long>(part) * C::kRows + 8 * r + 2 * c + e) * 2;
          ml[0] = top[r][e];
          ml[1] = sum[r][e] * fp8_pow2(-kHeadroom);  // (as the join takes it; the outputs have 2^kHeadroomLag as the sum)
        }
      }
      // products j: rows g and g + 8 are channels g D/8 + 2j and + 1
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + 8 * r + 2 * c + e;
        if (row >= p.rows) continue;
        if (whole) {
          const float inv = sum[r][e] == 0.f ? 0.f : 1.f / sum[r][e];
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

// Groups of eight query rows that one pass over the cache serves.
int row_groups(long long rows) { return rows <= 8 ? 1 : 2; }

// Rows from which on the 128-row tiles of the many-row kernel are the faster.  8 key/value heads and 65536
// tokens, us here and there: of 128 channels 32 rows 55 and 65, 48 rows 71 and 67, 128 rows 168 and 71; of 64 channels 39
// and 52, 53 and 53, 108 and 55; of 32 channels 31 and 50, 42 and 51, 80 and 53.  Where lengths differ much the tiles'
// ranges do, too (8 items, none to 16384 tokens each, 128 channels: 48 rows 74 and 110, 128 rows 178 and 117); over 2048
// tokens 17 rows are enough (16 and 15).  Lengths are on the device, so the rule has the rows alone.
constexpr long long kTileRows = 49;

template <int D, int G, typename T>
int launch(cudaStream_t stream, const AttnParams& p, unsigned int* status) {
  static unsigned long long configured = 0;
  int rc = ensure_smem_attribute(reinterpret_cast<const void*>(kv_int4_attention_kernel<D, G, T>),
                                 Cfg<D, G>::kOffBase + (kMaxBatch + 1) * 4, &configured, "kv_attention shared memory");
  if (rc != LDB_OK) return rc;
  rc = launch_kernel(kv_int4_attention_kernel<D, G, T>, dim3(p.warps / kWarps), dim3(kWarps * 32),
                     Cfg<D, G>::kOffBase + (p.c.batch + 1) * 4, stream, "kv_attention launch", p, status);
  return rc != LDB_OK ? rc : launch_merge<D, T>(stream, p, kTile);
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

int ldb_kv_attention_int4_workspace_size(int batch, int queries, int heads, int kv_heads, int head_dim,
                                         long long capacity, size_t* bytes) {
  using namespace ldb;
  if (!bytes) return fail(LDB_ERR_INVALID, "kv_attention: bytes is null");
  if (batch < 0 || queries < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads ||
      (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return fail(LDB_ERR_SHAPE, "kv_attention: %d heads over %d of width %d (32, 64 or 128)", heads, kv_heads, head_dim);
  const long long rows = static_cast<long long>(queries) * (heads / kv_heads);
  const int groups = row_groups(rows);
  *bytes = rows >= kTileRows
               ? kv_int4_tile_workspace(batch, kv_heads, rows, head_dim, capacity)
               : workspace_bytes_of(ctas_of(head_dim, groups) * sm_count() * kWarps, kGroupRows * groups, head_dim);
  return LDB_OK;
}

int ldb_kv_attention_int4(cudaStream_t stream, const ldb_kv_attention_desc* desc) {
  using namespace ldb;
  if (const int rc = check_desc(desc, "kv_attention")) return rc;
  const auto& [struct_size, dtype, cache, q, out, q_ld, q_batch, out_ld, out_batch, lengths, workspace, workspace_bytes,
               queries, heads, causal, scale] = *desc;
  const auto& [k_codes, v_codes, k_scales, v_scales, table, table_ld, pages, kv_heads, page, head_dim, width, batch] =
      cache;
  if (dtype != LDB_F16 && dtype != LDB_BF16) return fail(LDB_ERR_INVALID, "kv_attention: queries must be f16 or bf16");
  // (a NaN would not reach the rows: factors are kept above zero by a maximum)
  if (!std::isfinite(scale * 1.4426950408889634f))
    return fail(LDB_ERR_INVALID, "kv_attention: scale %g (finite, as a power of two's factor too)", scale);
  size_t need = 0;
  int rc = ldb_kv_attention_int4_workspace_size(batch, queries, heads, kv_heads, head_dim,
                                                static_cast<long long>(std::max(width, 0)) * std::max(page, 0), &need);
  if (rc != LDB_OK) return rc;
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return fail(LDB_ERR_SHAPE, "kv_attention: pages of %d tokens (16, 32, 64 or 128)", page);
  if (pages <= 0 || width <= 0 || table_ld < width || static_cast<long long>(width) * page > 0x7FFFFF00ll)
    return fail(LDB_ERR_SHAPE, "kv_attention: %d pages, table of %d", pages, width);
  if (static_cast<long long>(pages) * kv_heads > 0x7FFFFFFFll / page)
    return fail(LDB_ERR_SHAPE, "kv_attention: cache of %d pages, %d heads and %d tokens (2^31 - 1 rows)", pages, kv_heads, page);
  if (batch > kMaxBatch) return fail(LDB_ERR_SHAPE, "kv_attention: at most %d items, got %d", kMaxBatch, batch);
  if (batch == 0 || queries == 0) return LDB_OK;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !table || !lengths || !out)
    return fail(LDB_ERR_INVALID, "kv_attention: null pointer");
  const long long row = static_cast<long long>(heads) * head_dim;
  if ((queries > 1 && (q_ld < row || out_ld < row)) || (batch > 1 && out_batch < row))
    return fail(LDB_ERR_SHAPE, "kv_attention: a row stride, or the output's item stride, is below %lld", row);
  for (const uint8_t* t : {k_codes, v_codes, k_scales, v_scales})
    if (reinterpret_cast<uintptr_t>(t) % 16)
      return fail(LDB_ERR_ALIGNMENT, "kv_attention: codes and scales must be 16-byte aligned");
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
    return kv_int4_attention_tiles(stream, t, head_dim, dtype, scale, workspace, status);
  }
  AttnParams p{};
  p.c = view;
  p.q = q, p.q_ld = q_ld, p.q_batch = q_batch, p.q_vec = q_vec;
  p.out = out, p.out_ld = out_ld, p.out_batch = out_batch, p.out_vec = out_vec;
  p.queries = queries, p.group = heads / kv_heads;
  p.tile_rows = kGroupRows * row_groups(group_rows);
  const long long row_tiles = (group_rows + p.tile_rows - 1) / p.tile_rows;
  const long long tiles = kStart + (static_cast<long long>(width) * page + kTile - 1) / kTile;
  if (row_tiles * kv_heads * batch > 0x7FFFFFFFll / tiles)
    return fail(LDB_ERR_SHAPE, "kv_attention: too many heads over too long a table");
  p.rows = static_cast<int>(group_rows), p.row_tiles = static_cast<int>(row_tiles);
  p.causal = causal != 0;
  p.negate = scale < 0.f;
  p.scale_log2 = (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  p.warps = ctas_of(head_dim, row_groups(group_rows)) * sm_count() * kWarps;
  p.o_part = static_cast<float*>(workspace);
  p.ml_part = p.o_part + static_cast<size_t>(p.warps) * 2 * p.tile_rows * head_dim;
  p.open_by_pair = row_tiles * kv_heads * batch <= p.warps;
  p.status = status;
  p.open_part = reinterpret_cast<int4*>(p.ml_part + static_cast<size_t>(p.warps) * 2 * p.tile_rows * 2);
  return dtype == LDB_F16 ? launch_dim<__half>(stream, p, head_dim, status)
                          : launch_dim<__nv_bfloat16>(stream, p, head_dim, status);
}

}  // extern "C"
