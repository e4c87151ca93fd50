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
// two (exact down to 2^-17 of the row's largest).  Weights are rounded to f16 once, 2^15 at
// M and lost below 2^-40 of it; their sum is FP32.
//
// Bound: HBM, (D / 2 + D / 16) 2 bytes a token and key/value head, read once for
// a group's heads.  The tiles of 64 tokens of all items and heads form one line that the
// warps share out equally (kv_attention_ranges.cuh); a warp copies the next
// tiles into its own ring (cp.async) while it works on one.

#include <algorithm>

#include "host_common.h"
#include "kv_attention.cuh"
#include "kv_attention_ranges.cuh"
#include "kv_int4.cuh"
#include "kv_int4_attention.cuh"

namespace ldb {
namespace {

constexpr int kTile = 64;      // tokens per tile
constexpr int kGroupRows = 8;  // query rows of one value product
// Positions on the line that the start of a pair counts for.
constexpr int kStart = 2;
constexpr int kScaleRow = kTile + 16;  // bytes of a group's scales of a tile (padded: other banks for the next group)

// G groups of eight query rows per row tile.
template <int D, int G>
struct Cfg {
  static constexpr int kRows = G * kGroupRows;
  static constexpr int kTokenBytes = D / 2;
  static constexpr int kGroups = D / kInt4Group;
  static constexpr int kCodeBytes = kTile * kTokenBytes;
  static constexpr int kScaleBytes = kGroups * kScaleRow;
  static constexpr int kOffScale = 2 * kCodeBytes;  // in a slot: codes of K and V, then scales of K and V
  static constexpr int kSlotBytes = 2 * (kCodeBytes + kScaleBytes);
  static constexpr int kSlots = D == 128 ? 3 : (D == 64 ? 4 : 8);
  static constexpr int kCtasPerSm = D == 128 ? 2 : 3;
  static constexpr int kOffBase = kWarps * kSlots * kSlotBytes;  // [batch + 1] int
};
int ctas_per_sm(int head_dim) { return head_dim == 128 ? Cfg<128, 1>::kCtasPerSm : Cfg<64, 1>::kCtasPerSm; }

// A run of tiles of one (item, head, row tile) pair, and the copies of its tiles into the warp's ring.
template <int D>
struct Fetch {
  using C = Cfg<D, 1>;
  const KvView& c;
  int b, head, used;  // pages that hold the item's tokens
  int batch0;         // first of the 32 pages whose numbers the lanes hold
  int id;
  uint32_t holes;     // four bits a slot: 16 tokens of a page that the table names wrongly
  unsigned int* status;

  __device__ __forceinline__ Fetch(const KvView& view, unsigned int* st) : c(view), holes(0), status(st) {}

  __device__ __forceinline__ void start(int item, int h, int len) {
    b = item;
    head = h;
    used = (len + c.page - 1) / c.page;
    batch0 = -64;
  }

  // Copy tile j into slot `slot` of the ring at `ring` (shared address).
  __device__ __forceinline__ void tile(int j, uint32_t ring, int slot) {
    const uint32_t dst = ring + slot * C::kSlotBytes;
    const int lane = lane_id();
    const int shift = 31 - __clz(c.page);
    const int first = (j * kTile) >> shift;
    if (first - batch0 > 28) {  // (a tile has up to four pages)
      batch0 = first;
      const int at = batch0 + lane;
      id = at < used ? c.table[b * c.table_ld + at] : -1;
      if (at < used && (id < 0 || id >= c.pages)) {
        set_bad_shape(status);
        id = -1;
      }
    }
    // the page of each 16 tokens, and where in it they start
    int ids[4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      ids[n] = __shfl_sync(0xffffffffu, id, (((j * kTile) + 16 * n) >> shift) - batch0);
    holes &= ~(15u << (4 * slot));
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (ids[n] < 0) holes |= 1u << (4 * slot + n);
    const int inside = (j * kTile) & (c.page - 1);
    auto chunk_row = [&](int n) { return (inside + 16 * n) & (c.page - 1); };
    constexpr int kUnits = 16 * C::kTokenBytes / 16;  // 16-byte units of 16 tokens' codes: D / 2
#pragma unroll
    for (int i = 0; i < 4 * kUnits / 32; ++i) {
      const int u = i * 32 + lane;
      const int n = kUnits >= 32 ? i * 32 / kUnits : u / kUnits;
      const int page_id = kUnits >= 32 ? ids[n & 3] : ((n & 1) ? ids[(2 * i + 1) & 3] : ids[(2 * i) & 3]);
      const long long off =
          ((static_cast<long long>(max(page_id, 0)) * c.kv_heads + head) * c.page + chunk_row(n)) * C::kTokenBytes +
          (u % kUnits) * 16;
      const uint32_t bytes = page_id < 0 ? 0u : 16u;  // zeros for what has no page
      cp_async16(dst + u * 16, c.k + off, bytes);
      cp_async16(dst + C::kCodeBytes + u * 16, c.v + off, bytes);
    }
    // Scales: 16 tokens of one group a unit; K's and V's side by side over the lanes where they fit.
    {
      const int n = lane & 3;
      const int page_id = (n & 2) ? ((n & 1) ? ids[3] : ids[2]) : ((n & 1) ? ids[1] : ids[0]);
      const uint32_t bytes = page_id < 0 ? 0u : 16u;
      const long long unit = static_cast<long long>(max(page_id, 0)) * c.kv_heads + head;
      const uint32_t to = dst + C::kOffScale;
      if constexpr (D == 128) {
        const int group = lane >> 2;
        const long long off = (unit * C::kGroups + group) * c.page + chunk_row(n);
        cp_async16(to + group * kScaleRow + n * 16, c.k_scale + off, bytes);
        cp_async16(to + C::kScaleBytes + group * kScaleRow + n * 16, c.v_scale + off, bytes);
      } else {
        const int which = lane / (4 * C::kGroups), group = (lane >> 2) % C::kGroups;
        const long long off = (unit * C::kGroups + group) * c.page + chunk_row(n);
        if (which < 2)
          cp_async16(to + which * C::kScaleBytes + group * kScaleRow + n * 16, (which ? c.v_scale : c.k_scale) + off,
                     bytes);
      }
    }
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

  // Lane (g, c) holds, in q k, query row g of each group, channels [c D/4, (c + 1) D/4)
  // of the key in column g of each of eight products, and the scores of the keys
  // in columns 2c and 2c + 1; in p v, the tokens of those scores, the channels
  // [g D/8, (g + 1) D/8), and their outputs for rows 2c and 2c + 1.  Column j of
  // product n is token 16 (j / 2) + 2n + (j % 2, the other way round for odd j / 2): so a
  // lane's tokens in p v are 16 neighbours, whose scales are one 16-byte read, and no
  // eight (four) lanes that read at a time meet in a bank more than once (twice).
  const int g = lane >> 2, c = lane & 3;
  constexpr int kSteps = D / 16;            // q k products over the channels
  constexpr int kMTiles = D / 16;           // p v products over the channels
  constexpr int kWk = D / 8;                // bytes of a key's channels: 16, 8 or 4
  constexpr int kWv = D / 16;               // bytes of a value's: 8, 4 or 2
  const int odd_k = (g & 1) ^ ((g >> 1) & 1), odd_v = c & 1;
  const int at_k = (16 * (g >> 1) + odd_k) * C::kTokenBytes + c * kWk;
  const int at_v = C::kCodeBytes + 16 * c * C::kTokenBytes + g * kWv;
  const int at_ks = C::kOffScale + (c * (D / 4) / kInt4Group) * kScaleRow + 16 * (g >> 1);
  const int at_vs = C::kOffScale + C::kScaleBytes + (g * (D / 8) / kInt4Group) * kScaleRow + 16 * c;
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
      if (t < tiles) fetch.tile(tile0 + t, ring, t);
      cp_async_commit();
    }

    // Queries in the channel order of the unpacked keys, and their rows' factors.
    uint32_t qa[G][kSteps][2];
    float factor[G];
#pragma unroll
    for (int r = 0; r < G; ++r) {
      // a NaN stays one, an infinity makes the row's factor one
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < D / 8; ++k) {
        const float2 x = kv_unpack2<T>(raw[r][k]);
        m = fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y)));
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const int e = kv_query_exponent(m);
      factor[r] = (fp8_is_finite(m) ? (kScaled ? fp8_pow2(e - 7) * 0.0078125f : 1.f) : fp8_nan()) * p.scale_log2;
      if constexpr (kScaled) {
        const float inv = fp8_pow2(7 - e);  // largest magnitude to [2^7, 2^8), and then to [2^14, 2^15)
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          const float2 x = kv_unpack2<T>(raw[r][k]);
          raw[r][k] = pack_half2(x.x * inv * 128.f, x.y * inv * 128.f);
        }
      }
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
    float top[G], sum[G];
#pragma unroll
    for (int r = 0; r < G; ++r) top[r] = kFloor, sum[r] = 0.f;

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
      const uint32_t holes = fetch.holes >> (4 * slot) & 15u;
      const bool masked = j0 + kTile > open || holes;

      // Scores, eight keys at a time.
      float s[G][8][2];
      {
        constexpr int kKeyGroups = D == 128 ? 2 : 1;  // of the lane's channels
        uint32_t scales[kKeyGroups][4];
#pragma unroll
        for (int h = 0; h < kKeyGroups; ++h) lds_words<16>(sk + at_ks + h * kScaleRow, scales[h]);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          uint32_t w[kWk / 4];
          lds_words<kWk>(sk + at_k + 2 * n * C::kTokenBytes, w);
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kWk / 4; ++i) {
            const uint32_t sc = scale_pair(scales[kKeyGroups == 2 ? i >> 1 : 0][n >> 1], sel_k[n & 1]);
            uint32_t v[4];
            unpack4(w[i], as_half2(sc), minus72(sc), v);
#pragma unroll
            for (int h = 0; h < 2; ++h)
              mma_f16(d, qa[0][2 * i + h][0], G > 1 ? qa[G - 1][2 * i + h][0] : 0u, qa[0][2 * i + h][1],
                      G > 1 ? qa[G - 1][2 * i + h][1] : 0u, v[2 * h], v[2 * h + 1]);
          }
#pragma unroll
          for (int r = 0; r < G; ++r) {
            s[r][n][0] = d[2 * r] * factor[r];
            s[r][n][1] = d[2 * r + 1] * factor[r];
          }
        }
      }
      uint32_t vs[4];  // scales of the values of the lane's 16 tokens
      lds_words<16>(sk + at_vs, vs);
      uint64_t bad = 0;  // tokens whose values are NaN in the lane's group, where some rows may not see them
      if (masked) {
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tok = 16 * c + 2 * n + (e ^ odd_v);
#pragma unroll
            for (int r = 0; r < G; ++r)
              if (j0 + tok >= limit[r] || (holes >> c & 1u)) s[r][n][e] = -INFINITY;
          }
        const int left = len - j0 - 16 * c;  // of the lane's tokens, those that exist
        uint32_t mine = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
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
        bad = static_cast<uint64_t>(mine) << (16 * c);
        bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
        bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
      }
      float mx[G];
      bool grew = false;
#pragma unroll
      for (int r = 0; r < G; ++r) {
        mx[r] = kFloor;
#pragma unroll
        for (int n = 0; n < 8; ++n) mx[r] = fmaxf(mx[r], fmaxf(s[r][n][0], s[r][n][1]));
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
      // Weights 2^(s - M + kHeadroom): the fragments of p v as they are.
      uint32_t pf[G][8];
#pragma unroll
      for (int r = 0; r < G; ++r) {
        const float ref = top[r] - kHeadroom;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float a = ex2_approx(s[r][n][0] - ref), bb = ex2_approx(s[r][n][1] - ref);
          sum[r] += a + bb;
          pf[r][n] = pack_half2(a, bb);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
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
            const int seen = __shfl_sync(0xffffffffu, limit[r], 8 * c + 4 * e) - j0;  // of the tile's tokens
            const uint64_t in = seen <= 0 ? 0 : (seen >= 64 ? ~0ull : (1ull << seen) - 1);
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
    const bool whole = tiles == item_tiles;
    const int part = me * 2 + (tile0 == 0 ? 1 : 0);
#pragma unroll
    for (int r = 0; r < G; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      if (!whole && c == 0) {
        float* ml = p.ml_part + (static_cast<long long>(part) * C::kRows + 8 * r + g) * 2;
        ml[0] = top[r];
        ml[1] = sum[r] * fp8_pow2(-kHeadroom);
      }
      const float l[2] = {__shfl_sync(0xffffffffu, sum[r], 8 * c), __shfl_sync(0xffffffffu, sum[r], 8 * c + 4)};
      // products j: rows g and g + 8 are channels g D/8 + 2j and + 1
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + 8 * r + 2 * c + e;
        if (row >= p.rows) continue;
        if (whole) {
          const float inv = l[e] == 0.f ? 0.f : 1.f / l[e];
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

// Rows from which on the 128-row tiles of the many-row kernel are the faster.
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
  *bytes = rows >= kTileRows ? kv_int4_tile_workspace(batch, kv_heads, rows, head_dim, capacity)
                             : workspace_bytes_of(ctas_per_sm(head_dim) * sm_count() * kWarps,
                                                  kGroupRows * row_groups(rows), head_dim);
  return LDB_OK;
}

int ldb_kv_attention_int4(cudaStream_t stream, const void* q, long long q_ld, long long q_batch, int dtype,
                          const uint8_t* k_codes, const uint8_t* v_codes, const uint8_t* k_scales,
                          const uint8_t* v_scales, int pages, int kv_heads, int page, int head_dim, const int* table,
                          long long table_ld, int width, const int* lengths, void* out, long long out_ld,
                          long long out_batch, int batch, int queries, int heads, float scale, int causal,
                          void* workspace, size_t workspace_bytes) {
  using namespace ldb;
  if (dtype != LDB_F16 && dtype != LDB_BF16) return fail(LDB_ERR_INVALID, "kv_attention: queries must be f16 or bf16");
  size_t need = 0;
  int rc = ldb_kv_attention_int4_workspace_size(batch, queries, heads, kv_heads, head_dim,
                                                static_cast<long long>(std::max(width, 0)) * std::max(page, 0), &need);
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
