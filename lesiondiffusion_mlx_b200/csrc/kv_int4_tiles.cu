// Attention of many query rows over the paged 4-bit key/value cache, on the
// tcgen05 tensor cores (few rows: kv_int4_attention.cu, whose formulas these are).
//
// One CTA owns two 128-row tiles of one (item, key/value head) and streams
// blocks of 128 tokens once for both.  Keys and values become f16 (exact) on the way: a
// warp reads a token a lane from the cache into registers, a piece of 32 tokens ahead,
// unpacks it and writes its row to shared memory as the products read it.
// Unpacking leaves eight channels in the order 0, 4, 1, 5, 2, 6, 3, 7: the queries
// are laid out alike, and an output row is put in order as it leaves.  Queries are f16
// as they are, or bf16 rows scaled by a power of two.  The weights are f16 in TMEM, 2^7 at the row's
// reference, which may lag 2^8 behind its maximum: 11 bits down to 2^-21 of the
// reference, nothing below 2^-32.
//
// Warps: 0 issues the products, 1-7 unpack, 8-15 and 16-23 run the online softmax of
// tile 0 and 1, half a row a thread.  Grids that leave SMs idle cut the tokens into ranges, merged
// by a second kernel (kv_attention_tiles.cuh).
//
// Bound: 4 D flops and one exponential per score.  One B200, 1024 causal bf16 queries of 2 items, 32 heads of
// 128 over 8, behind 8192 and 16384 tokens: 458 us (862 TFLOP/s), some 4400 cycles a block on SMs that share 256 CTAs out
// unevenly; the products need 2048 of them and read 128 bytes of shared memory a cycle all the while.  6400 f16
// queries of 4 heads of 64 over 6477 tokens 118 us, some 4060 cycles a block for 2048 of exponentials.  Each tile is a
// chain: scores, weights (1500 cycles alone, 1024 of them exponentials), votes, value product.  (Cycles of the kernel without
// far references, 2 % faster.  At 80 registers a thread two tiles of 128 channels spill 20 bytes, narrower ones 12 and
// alternating ones none.)  Slower or no faster, the first case's us, where it took 443: one row a thread with four unpacking warps (485) or seven (583); two
// issuing warps (637); packed rows through a ring of cp.async (606); blocks of 64 keys with two places for each tile's scores
// (476: products of 64 columns read the queries twice); the tiles' weights in strict turn (498); maxima before weights, scores
// read from TMEM twice (481); the line of all blocks cut in equal ranges (508); polynomial exponentials.

#include <algorithm>

#include "host_common.h"
#include "kv_attention.cuh"
#include "kv_attention_tiles.cuh"
#include "kv_int4.cuh"
#include "kv_int4_attention.cuh"

namespace ldb {
namespace {

constexpr int kThreads = 768;     // of 80 registers: a row's scores are shared by two threads
constexpr int kUnpackWarps = 7;
constexpr int kMeta = 4;          // ring of the masks of missing pages

template <int D>
struct Cfg {
  static constexpr int kSubD = D == 32 ? 32 : 64;  // channels of one swizzled tile
  static constexpr int kSubRow = kSubD * 2;
  static constexpr uint32_t kLayout = kSubD == 64 ? kSwizzle128 : kSwizzle64;
  static constexpr int kTileBytes = kN * D * 2;    // 128 rows: queries, keys or values
  static constexpr int kGroups = D / kInt4Group;
  static constexpr int kOffK = 2 * kTileBytes;
  static constexpr int kOffV = kOffK + 2 * kTileBytes;
  static constexpr int kOffMeta = kOffV + 2 * kTileBytes;  // [kMeta][4] bytes: a bit for each 16 tokens of a missing page
  static constexpr int kOffBad = kOffMeta + kMeta * 4;     // NaN met among values that not every row sees
  static constexpr int kOffVote = kOffBad + 16;            // [8 pairs of warps][2][half]: a reference has to grow
  static constexpr int kOffRow = kOffVote + 128;           // [tile][half][kM] floats that a row's two threads exchange
  static constexpr int kOffBar = kOffRow + 4 * kM * 4;
  static constexpr int kSmem = 1024 + kOffBar + 320;
  // TMEM: S_t at 128 t, O_t at 256 + 128 t.  D = 128: the weights overwrite
  // their scores; narrower heads have room for them behind O_t, so that the next block's
  // scores need not wait for the value product.
  static constexpr bool kSeparateP = D <= 64;
  static_assert(kSmem <= 232448, "shared memory");
  // Where 16 bytes (channels 8 chunk ..) of a row lie in a tile.
  static __device__ __forceinline__ int place(int row, int chunk) {
    constexpr int kPer = kSubRow / 16;
    return (chunk / kPer) * kN * kSubRow + swizzle_offset(row * kSubRow + (chunk % kPer) * 16, kSubRow);
  }
};

// D[tmem] (+)= A[smem] * B[smem]^T of f16 operands, by one elected lane of a convergent warp.
__device__ __forceinline__ void umma_ss_warp(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// A score of minus infinity where `at` >= `seen`, or where a bit of `mask` is set.  Volatile with the
// comparison inside, so that blocks without hidden keys branch around them.
__device__ __forceinline__ void hide_from(uint32_t& score, int at, int seen) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.s32 p, %1, %2;\n\t@p mov.b32 %0, 0xFF800000;\n\t}\n"
               : "+r"(score)
               : "r"(at), "r"(seen));
}
__device__ __forceinline__ void hide_if(uint32_t& score, uint32_t mask, uint32_t bit) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 m;\n\tand.b32 m, %1, %2;\n\tsetp.ne.u32 p, m, 0;\n\t"
      "@p mov.b32 %0, 0xFF800000;\n\t}\n"
      : "+r"(score)
      : "r"(mask), "r"(bit));
}

// Wait for the loads from TMEM; what uses these registers comes after.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// A token's codes and scales of keys or of values.
template <int D>
struct Packed {
  uint4 code[D / 32];
  uint32_t scale[D / kInt4Group];  // (a byte each: put together they would be waited for where they are loaded)
};

// ALT: one tile of rows, alternating: tile t is the rows over the blocks of parity t, so that the softmax of one block
// runs beside the products of the next; each leaves its part for the merge.
template <int D, typename T, bool ALT>
__global__ void __launch_bounds__(kThreads, 1) kv_int4_tiles_kernel(const KvTileParams p, unsigned int* status) {
  using C = Cfg<D>;
  constexpr bool kScaled = !std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_meta = smem + C::kOffMeta;
  uint32_t* s_bad = reinterpret_cast<uint32_t*>(smem + C::kOffBad);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;              // the queries are written
  uint64_t* k_full = q_full + 1;        // [2] f16 keys are written
  uint64_t* k_empty = k_full + 2;       // [2] both tiles' scores have read them
  uint64_t* v_full = k_empty + 2;       // [2] f16 values are written
  uint64_t* v_empty = v_full + 2;       // [2] the value products have read them
  uint64_t* meta_full = v_empty + 2;    // [kMeta] the mask of missing pages is written
  uint64_t* s_full = meta_full + kMeta; // [2] per tile
  uint64_t* s_free = s_full + 2;        // [2] scores are in registers
  uint64_t* p_ready = s_free + 2;       // [2] weights are in TMEM
  uint64_t* pv_done = p_ready + 2;      // [2]
  uint64_t* pair_bar = pv_done + 2;     // [8] the two warps of 32 rows meet
  uint64_t* drain = pair_bar + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((1 + 8 + kMeta + 8 + 8 + 1) * 8 + 8 <= 320, "barrier block");

  const int warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    mbar_init(drain, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 4);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 8);
      mbar_init(&p_ready[s], 8);
      mbar_init(&pv_done[s], 1);
    }
    for (int s = 0; s < kMeta; ++s) mbar_init(&meta_full[s], 4);
    for (int s = 0; s < 8; ++s) mbar_init(&pair_bar[s], 2);
    mbar_init(q_full, ALT || p.rows - (p.row_blocks - 1 - static_cast<int>(blockIdx.x) / p.splits) * 2 * kM > kM ? 16 : 8);
    *abort_flag = 0;
    *s_bad = 0;
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_begin();
  const Span sp = span_of(p, status);

  if (warp == 0) {
    if (sp.nblocks > 0) {
      // --------------------------------------------------------- products
      constexpr uint32_t idesc_qk = make_idesc_f16(kM, kN, 0u, 0u, 0u);
      constexpr uint32_t idesc_pv = make_idesc_f16(kM, D, 0u, 0u, 1u);
      auto scores = [&](int t, int j) {
        const uint32_t q_addr = smem_u32(smem + t * C::kTileBytes);
        const uint32_t k_addr = smem_u32(smem + C::kOffK + (j & 1) * C::kTileBytes);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k * 16 / C::kSubD) * kN * C::kSubRow + (k * 32) % C::kSubRow;
          umma_ss_warp(tmem + t * 128, make_smem_desc(q_addr + off, 16, 8 * C::kSubRow, C::kLayout),
                       make_smem_desc(k_addr + off, 16, 8 * C::kSubRow, C::kLayout), idesc_qk, k > 0 ? 1u : 0u);
        }
        umma_commit_warp(&s_full[t]);
      };
      auto values = [&](int t, int j) {
        const uint32_t v_addr = smem_u32(smem + C::kOffV + (j & 1) * C::kTileBytes);
        // weights of the keys' second half: over their own scores, too
        const uint32_t p_tmem = C::kSeparateP ? tmem + 256 + t * 128 + 64 : tmem + t * 128;
#pragma unroll
        for (int k = 0; k < kN / 16; ++k)  // (tiles of 64 channels lie kN rows apart)
          umma_ts_warp(tmem + 256 + t * 128, p_tmem + k * 8 + (C::kSeparateP || k < 4 ? 0 : 32),
                       make_smem_desc(v_addr + k * 16 * C::kSubRow, kN * C::kSubRow, 8 * C::kSubRow, C::kLayout),
                       idesc_pv, (j > (ALT ? 1 : 0) || k > 0) ? 1u : 0u);
        umma_commit_warp(&pv_done[t]);
      };
      bool ok = warp_wait(q_full, 0, abort_flag, status);
      // (the blocks that tile j & 1 has had before block j are j >> 1)
      for (int j = 0; ALT && ok && j < sp.nblocks + (C::kSeparateP ? 1 : 2); ++j) {
        const int t = j & 1, last = C::kSeparateP ? j - 1 : j - 2;  // of the value product
        auto value_product = [&] {
          if (last < 0) return;
          ok = warp_wait(&v_full[last & 1], static_cast<uint32_t>(last >> 1) & 1u, abort_flag, status) &&
               warp_wait(&p_ready[last & 1], static_cast<uint32_t>(last >> 1) & 1u, abort_flag, status);
          if (!ok) return;
          tc_fence_after();
          values(last & 1, last);
          umma_commit_warp(&v_empty[last & 1]);
        };
        if (!C::kSeparateP) value_product();
        if (ok && j < sp.nblocks) {
          ok = warp_wait(&k_full[t], static_cast<uint32_t>(j >> 1) & 1u, abort_flag, status) &&
               (!C::kSeparateP || j < 2 || warp_wait(&s_free[t], static_cast<uint32_t>((j >> 1) - 1) & 1u, abort_flag, status));
          if (!ok) break;
          tc_fence_after();
          scores(t, j);
          umma_commit_warp(&k_empty[t]);
        }
        if (ok && C::kSeparateP) value_product();
      }
      for (int j = 0; !ALT && ok && j <= sp.nblocks; ++j) {
        const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u, was = static_cast<uint32_t>(j - 1) & 1u;
        if (j < sp.nblocks) ok = warp_wait(&k_full[j & 1], ph, abort_flag, status);
        if (ok && j > 0)
          ok = warp_wait(&v_full[(j - 1) & 1], static_cast<uint32_t>((j - 1) >> 1) & 1u, abort_flag, status);
        if constexpr (C::kSeparateP) {
          for (int t = 0; ok && j < sp.nblocks && t < sp.tiles; ++t) {
            // the softmax has the scores of the block before in registers
            if (j > 0) ok = warp_wait(&s_free[t], was, abort_flag, status);
            if (!ok) break;
            tc_fence_after();
            scores(t, j);
          }
          if (ok && j < sp.nblocks) umma_commit_warp(&k_empty[j & 1]);
          for (int t = 0; ok && j > 0 && t < sp.tiles; ++t) {
            ok = warp_wait(&p_ready[t], was, abort_flag, status);
            if (!ok) break;
            tc_fence_after();
            values(t, j - 1);
          }
        } else {
          for (int t = 0; ok && t < sp.tiles; ++t) {
            if (j > 0) {
              ok = warp_wait(&p_ready[t], was, abort_flag, status);
              if (!ok) break;
              tc_fence_after();
              values(t, j - 1);
            }
            if (j < sp.nblocks) {
              if (j == 0) tc_fence_after();
              scores(t, j);
            }
          }
          if (ok && j < sp.nblocks) umma_commit_warp(&k_empty[j & 1]);
        }
        if (ok && j > 0) umma_commit_warp(&v_empty[(j - 1) & 1]);
      }
      umma_commit_warp(drain);
      volatile int never = 0;
      mbar_wait(drain, 0, &never, status);
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ unpacking
    // Pieces of 32 tokens, a token per lane: four of the keys, then four of the values of each block, dealt out
    // in turn; a warp reads its next piece into registers while it unpacks one.
    const int shift = 31 - __clz(p.c.page);
    const int pieces = sp.nblocks * 8;
    // What the table says for the lane's token of piece n, kNone where it has none.  (Looked at a piece
    // later, when it is used: a test here would wait for it.)
    constexpr int kNone = -0x7FFFFFFF - 1;
    auto page_of = [&](int n) {
      const int tok = (sp.jb0 + (n >> 3)) * kN + (n & 3) * 32 + lane;
      return n < pieces && tok < sp.len ? p.c.table[sp.b * p.c.table_ld + (tok >> shift)] : kNone;
    };
    auto known = [&](int id) { return id >= 0 && id < p.c.pages; };
    auto load = [&](int n, int id, Packed<D>& to) {
      if (!known(id)) {  // zeros: codes are of no account under a scale of zero
#pragma unroll
        for (int i = 0; i < D / 32; ++i) to.code[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < C::kGroups; ++g) to.scale[g] = 0;
        return;
      }
      const int in = ((n & 3) * 32 + lane) & (p.c.page - 1);  // (a block starts a page, or 128 tokens are one)
      const long long unit = static_cast<long long>(id) * p.c.kv_heads + sp.head;
      const uint4* from =
          reinterpret_cast<const uint4*>((n & 4 ? p.c.v : p.c.k) + (unit * p.c.page + in) * (D / 2));
#pragma unroll
      for (int i = 0; i < D / 32; ++i) to.code[i] = from[i];
      const uint8_t* s = (n & 4 ? p.c.v_scale : p.c.k_scale) + unit * C::kGroups * p.c.page + in;
#pragma unroll
      for (int g = 0; g < C::kGroups; ++g) to.scale[g] = s[g * p.c.page];
    };
    Packed<D> now, next;
    int n = warp - 1, id = page_of(n), id_next = page_of(n + kUnpackWarps);
    load(n, id, now);
    for (; n < pieces; n += kUnpackWarps) {
      const int j = n >> 3, st = j & 1, ms = j % kMeta, quarter = n & 3;
      const bool values = n & 4;
      const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u;
      const int id_after = page_of(n + 2 * kUnpackWarps);
      load(n + kUnpackWarps, id_next, next);
      if (!warp_wait(values ? &v_empty[st] : &k_empty[st], ph ^ 1u, abort_flag, status)) break;
      if (values) {
        if ((sp.jb0 + j + 1) * kN > sp.open) {
          // Where some rows may not see a token its NaN becomes zero here, and
          // the rows that do see it get the NaN at the end.
#pragma unroll
          for (int g = 0; g < C::kGroups; ++g) {
            if (now.scale[g] == kInt4NanScale) {
              now.scale[g] = 0;
              *s_bad = 1;
            }
          }
        }
      } else {
        // (the scores of block j - 2 are done, so the softmax has read the mask of block j - 4)
        const bool lost = id != kNone && !known(id);
        if (lost) set_bad_shape(status);
        const uint32_t missing = __ballot_sync(0xffffffffu, lost);
        if (lane == 0) {
          s_meta[ms * 4 + quarter] = ((missing & 0xFFFFu) ? 1 : 0) | ((missing >> 16) ? 2 : 0);
          mbar_arrive(&meta_full[ms]);
        }
      }
      uint8_t* to = smem + (values ? C::kOffV : C::kOffK) + st * C::kTileBytes;
      const int row = quarter * 32 + lane;
#pragma unroll
      for (int g = 0; g < C::kGroups; ++g) {
        const uint32_t sc = now.scale[g] * 0x00800080u;  // twice as f16
        const __half2 m = minus72(sc);
        const uint4 w = now.code[g >> 1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[4];
          unpack4((g & 1) ? (h ? w.w : w.z) : (h ? w.y : w.x), as_half2(sc), m, v);
          *reinterpret_cast<uint4*>(to + C::place(row, 2 * g + h)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(values ? &v_full[st] : &k_full[st]);
      now = next;
      id = id_next;
      id_next = id_after;
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int t = (warp - 8) >> 3;         // tile
    const int half = (warp >> 2) & 1;      // keys 64 half .. of a block, channels D / 2 half .. of the output
    const int quarter = warp & 3;          // TMEM lanes this warp may access
    const int pair = t * 4 + quarter;      // with the warp of the other half
    const int local = quarter * 32 + lane;
    const int row = sp.row0 + (ALT ? 0 : t * kM) + local;
    const int blocks = ALT ? (sp.nblocks - t + 1) >> 1 : sp.nblocks;  // of the tile
    const bool live = row < p.rows;
    const int i = live ? row / p.group : 0, gq = live ? row % p.group : 0;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tmem_s = tmem + t * 128 + lane_base + 64 * half;
    const uint32_t tmem_o = tmem + 256 + t * 128 + lane_base;
    const uint32_t tmem_p = C::kSeparateP ? tmem_o + 64 + 32 * half : tmem_s;
    const int limit = p.causal && live ? min(sp.len, sp.len - p.queries + i + 1) : sp.len;  // keys that the row sees
    float* s_row = reinterpret_cast<float*>(smem + C::kOffRow) + t * 2 * kM + local;  // [half * kM]
    volatile uint32_t* s_vote = reinterpret_cast<volatile uint32_t*>(smem + C::kOffVote) + pair * 4;
    uint32_t meets = 0;
    bool ok = ALT || t < sp.tiles;
    // The two warps of the rows wait for each other; what either has written to shared memory before is there for the other.
    auto meet = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&pair_bar[pair]);
      ok = warp_wait(&pair_bar[pair], meets & 1u, abort_flag, status);
      ++meets;
    };
    constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // lanes of a row (eight channels each), rows at a time
    const T* src = static_cast<const T*>(p.q) + sp.b * p.q_batch + i * p.q_ld +
                   (static_cast<long long>(sp.head) * p.group + gq) * D;
    float factor = 1.f;
    if (ok && sp.nblocks > 0) {
      // Query rows in the keys' order of channels, half of them each warp; the largest magnitude of a bf16
      // row to [2^14, 2^15).  A NaN stays one, an infinity makes the row's factor one (of a row that
      // sees any key).
      const int part_lane = lane % kLanes;
      constexpr int kTurns = kLanes / 2, kAtOnce = kTurns < 4 ? kTurns : 4;
#pragma unroll 1
      for (int n0 = half * kTurns; n0 < (half + 1) * kTurns; n0 += kAtOnce) {
        uint4 raw[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          const int from = (n0 + n) * kRows + lane / kLanes;  // row of the warp, and the lane that owns it
          const T* at = reinterpret_cast<const T*>(__shfl_sync(
                            0xffffffffu, reinterpret_cast<unsigned long long>(src), from)) + 8 * part_lane;
          raw[n] = make_uint4(0, 0, 0, 0);
          if (row - lane + from < p.rows) {
            if (p.q_vec) {
              raw[n] = *reinterpret_cast<const uint4*>(at);
            } else {
              const uint16_t* h = reinterpret_cast<const uint16_t*>(at);
              raw[n] = make_uint4(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16,
                                  h[4] | static_cast<uint32_t>(h[5]) << 16, h[6] | static_cast<uint32_t>(h[7]) << 16);
            }
          }
        }
#pragma unroll
        for (int k4 = 0; k4 < kAtOnce; ++k4) {
          const int from = (n0 + k4) * kRows + lane / kLanes;
          uint32_t w[4] = {raw[k4].x, raw[k4].y, raw[k4].z, raw[k4].w};
          float m = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 x = kv_unpack2<T>(w[k]);
            m = fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          if (part_lane == 0) s_row[from - lane] = m;
          if constexpr (kScaled) {
            const float inv = fp8_pow2(7 - kv_query_exponent(m));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 x = kv_unpack2<T>(w[k]);
              w[k] = as_word(__floats2half2_rn(x.x * inv * 128.f, x.y * inv * 128.f));
            }
          }
          const uint32_t flip = p.negate ? 0x80008000u : 0u;
          const uint4 out = make_uint4(__byte_perm(w[0], w[2], 0x5410) ^ flip, __byte_perm(w[0], w[2], 0x7632) ^ flip,
                                       __byte_perm(w[1], w[3], 0x5410) ^ flip, __byte_perm(w[1], w[3], 0x7632) ^ flip);
          *reinterpret_cast<uint4*>(smem + t * C::kTileBytes + C::place(quarter * 32 + from, part_lane)) = out;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      meet();
      const float top_of = *s_row;  // largest magnitude of the thread's row
      factor = fp8_is_finite(top_of) || limit <= 0
                   ? (kScaled ? fp8_pow2(kv_query_exponent(top_of) - 7) * 0.0078125f : 1.f) * p.scale_log2
                   : fp8_nan();
      if (factor < 1.2e-38f) factor = 1.2e-38f;  // (-inf times zero would be a NaN)
      if (ok) meet();  // (s_row is free again)
    }
    float top = kUnseen, l = 0.f;
    const uint64_t f2 = pack2(factor, factor);
    // The first block's largest scores are the first reference.
    if (ok && blocks > 0) {
      ok = warp_wait(&s_full[t], 0, abort_flag, status) && warp_wait(&meta_full[ALT ? t : 0], 0, abort_flag, status);
      if (ok) {
        tc_fence_after();
        const uint32_t missing = *reinterpret_cast<const uint32_t*>(s_meta + (ALT ? t : 0) * 4) >> (16 * half);
        const int j0 = (sp.jb0 + (ALT ? t : 0)) * kN + 64 * half;
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t sr[32];
          tmem_ld32(tmem_s + 32 * c, sr);
          tmem_wait_ld32(sr);
          if (j0 + 64 > sp.open || missing) {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              hide_from(sr[k], 32 * c + k, limit - j0);
              hide_if(sr[k], missing, 1u << (8 * c + k / 16));
            }
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2)
            m4[(k >> 1) & 3] = max3(m4[(k >> 1) & 3], __uint_as_float(sr[k]), __uint_as_float(sr[k + 1]));
        }
        s_row[half * kM] = __fmul_rn(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), factor);
        meet();
        if (ok) top = fmaxf(top, fmaxf(s_row[0], s_row[kM]));
        if (ok) meet();  // (s_row is free again)
      }
    }
    for (int nth = 0; ok && nth < blocks; ++nth) {
      const int j = ALT ? 2 * nth + t : nth;
      ok = warp_wait(&s_full[t], static_cast<uint32_t>(nth) & 1u, abort_flag, status) &&
           warp_wait(&meta_full[j % kMeta], static_cast<uint32_t>(j / kMeta) & 1u, abort_flag, status);
      if (!ok) break;
      tc_fence_after();
      const uint32_t missing = *reinterpret_cast<const uint32_t*>(s_meta + (j % kMeta) * 4) >> (16 * half);
      const int j0 = (sp.jb0 + j) * kN + 64 * half;
      const bool hidden = j0 + 64 > sp.open || missing;
      uint32_t packed[32];
      uint64_t sum2[2];
      float mx;
      // Weights 2^(by s + kHeadroom - off), and the thread's largest score.
      auto weights = [&](uint64_t by, float off) {
        const uint64_t shift = pack2(kHeadroom - off, kHeadroom - off);
        sum2[0] = sum2[1] = 0;
        mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t sr[32];
          tmem_ld32(tmem_s + 32 * c, sr);
          tmem_wait_ld32(sr);
          if (hidden) {  // hidden keys count nothing, nor do those of missing pages
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              hide_from(sr[k], 32 * c + k, limit - j0);
              hide_if(sr[k], missing, 1u << (8 * c + k / 16));
            }
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            mx = max3(mx, __uint_as_float(sr[k]), __uint_as_float(sr[k + 1]));
            float x0, x1;
            unpack2(fma2(pack2(__uint_as_float(sr[k]), __uint_as_float(sr[k + 1])), by, shift), x0, x1);
            const float e0 = ex2_approx(x0), e1 = ex2_approx(x1);
            sum2[(k >> 1) & 1] = add2(sum2[(k >> 1) & 1], pack2(e0, e1));
            packed[16 * c + k / 2] = as_word(__floats2half2_rn(e0, e1));
          }
        }
      };
      weights(f2, top);  // (against the reference as it is)
      // A reference seldom grows; where one of 32 rows' does, both warps scale what there is and begin again (as they do
      // wherever one is far).
      const bool mine =
          __any_sync(0xffffffffu, __fmul_rn(mx, factor) > (fabsf(top) > kFarReference ? -INFINITY : top + kGrow));
      const uint32_t side = (meets & 1u) * 2;
      if (lane == 0) s_vote[side + half] = mine;
      meet();
      if (!ok) break;
      if (mine || s_vote[side + 1 - half]) {
        s_row[half * kM] = __fmul_rn(mx, factor);
        meet();
        if (!ok) break;
        const float all = fmaxf(s_row[0], s_row[kM]);
        const float next = all - top > kGrow ? all : top;
        const float scale_half = ex2_approx(0.5f * (top - next)), alpha = scale_half * scale_half;
        if (nth > 0) {
          // the value product of the block before is done: the output is whole
          ok = warp_wait(&pv_done[t], static_cast<uint32_t>(nth - 1) & 1u, abort_flag, status);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < D / 2; c0 += 16) {
            uint32_t r[16];
            tmem_ld16(tmem_o + half * (D / 2) + c0, r);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * alpha);
            tmem_st16(tmem_o + half * (D / 2) + c0, r);
          }
          tmem_wait_st();
        }
        l = kv_scaled(l, scale_half);
        top = next;
        const bool far = __any_sync(0xffffffffu, is_far(top));
        if (far) {
          // (rare) What is above the references takes the scores' place.
#pragma unroll 1
          for (int c = 0; c < 64; c += 16) {
            uint32_t r[16];
            tmem_ld16(tmem_s + c, r);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__fmul_rn(__uint_as_float(r[k]), factor) - top);
            tmem_st16(tmem_s + c, r);
          }
          tmem_wait_st();
        }
        const float by = far ? 1.f : factor;
        weights(pack2(by, by), far ? 0.f : top);
        meet();  // (s_row is free again)
        if (!ok) break;
      }
      float a, b;
      unpack2(add2(sum2[0], sum2[1]), a, b);
      l += a + b;
      if constexpr (C::kSeparateP) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t]);
        if (nth > 0) {
          // the value product of the block before has read its weights
          ok = warp_wait(&pv_done[t], static_cast<uint32_t>(nth - 1) & 1u, abort_flag, status);
          if (!ok) break;
          tc_fence_after();
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_st16(tmem_p + 16 * c, *reinterpret_cast<uint32_t(*)[16]>(&packed[16 * c]));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t]);
    }
    if (ok && blocks > 0) {
      const int j = ALT ? 2 * (blocks - 1) + t : blocks - 1;
      ok = warp_wait(&pv_done[t], static_cast<uint32_t>(blocks - 1) & 1u, abort_flag, status) &&
           warp_wait(&v_full[j & 1], static_cast<uint32_t>(j >> 1) & 1u, abort_flag, status);  // (done as well: orders the reads of s_bad)
    }
    if (ALT) asm volatile("bar.sync 1, 512;" ::: "memory");  // (and those of the other tile's blocks)
    if (ok) {
      s_row[half * kM] = l;
      meet();
    }
    if (ok) {
      tc_fence_after();
      l = s_row[0] + s_row[kM];
      const bool parts = ALT || p.splits > 1;
      const int split = ALT ? 2 * (blockIdx.x % p.splits) + t : blockIdx.x % p.splits;
      const long long part =
          ((static_cast<long long>(split) * p.c.batch + sp.b) * p.c.kv_heads + sp.head) * p.rows + row;
      T* dst = static_cast<T*>(p.out) + sp.b * p.out_batch + i * p.out_ld +
               (static_cast<long long>(sp.head) * p.group + gq) * D;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // (one range: rows to shared memory, where the queries were, and from there D / 8 lanes a row)
      constexpr int kSpread = kLanes < 8 ? kLanes - 1 : 7;  // 16-byte pieces of an output row
      uint8_t* rows = smem + t * C::kTileBytes + quarter * 32 * D * 2;
      constexpr int kOrder[8] = {0, 2, 4, 6, 1, 3, 5, 7};  // where a channel of eight is
#pragma unroll 2
      for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 16) {
        uint32_t r[16];
        if (blocks > 0) {
          tmem_ld16(tmem_o + c0, r);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) r[c] = 0;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) x[c] = __uint_as_float(r[8 * h + kOrder[c]]);
          if (parts) {
            if (live) {
              float4* to = reinterpret_cast<float4*>(p.o_part + part * D + c0 + 8 * h);
              to[0] = make_float4(x[0], x[1], x[2], x[3]);
              to[1] = make_float4(x[4], x[5], x[6], x[7]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) x[c] *= inv;
            store8<T>(reinterpret_cast<T*>(rows + lane * D * 2 + ((c0 / 8 + h) ^ (lane & kSpread)) * 16), x);
          }
        }
        __syncwarp();  // the next read of TMEM is the whole warp's
      }
      if (!parts) {
        meet();
#pragma unroll 4
        for (int n = half * (kLanes / 2); ok && n < (half + 1) * (kLanes / 2); ++n) {
          const int from = n * kRows + lane / kLanes, chunk = lane % kLanes;
          T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), from)) +
                  8 * chunk;
          if (row - lane + from >= p.rows) continue;
          const uint4 v = *reinterpret_cast<const uint4*>(rows + from * D * 2 + (chunk ^ (from & kSpread)) * 16);
          if (p.out_vec) {
            *reinterpret_cast<uint4*>(to) = v;
          } else {
            const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int c = 0; c < 8; ++c) to[c] = e[c];
          }
        }
        __syncwarp();
      }
      if (parts && live && half == 0)
        *reinterpret_cast<float2*>(p.ml_part + part * 2) = make_float2(top, l * fp8_pow2(-kHeadroom));
      tc_fence_before();
      const bool bad = sp.nblocks > 0 && *s_bad != 0;  // (of the CTA: both warps go on or neither)
      if (bad && ok) meet();  // (the rows are written)
      if (bad && ok && live) {
        // Rare: NaN among the values of the blocks that `open` cuts, whose product
        // left them out.  Looked up again in the cache, token by token, by each row's threads.
        const int to = min(limit, (sp.jb0 + sp.nblocks) * kN);
        for (int tok = max(sp.jb0, max(sp.open, 0) / kN) * kN; tok < to; ++tok) {
          const int id = p.c.table[sp.b * p.c.table_ld + tok / p.c.page];
          if (id < 0 || id >= p.c.pages) continue;
          const uint8_t* s = p.c.v_scale +
                             (static_cast<long long>(id) * p.c.kv_heads + sp.head) * C::kGroups * p.c.page +
                             tok % p.c.page;
          for (int c = half * (D / 2); c < (half + 1) * (D / 2); ++c) {
            if (s[(c / kInt4Group) * p.c.page] != kInt4NanScale) continue;
            if (parts) {
              p.o_part[part * D + c] = fp8_nan();
            } else {
              dst[c] = from_f32<T>(fp8_nan());
            }
          }
        }
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, typename T, bool ALT>
int launch(cudaStream_t stream, KvTileParams p, unsigned int* status) {
  static unsigned long long configured = 0;
  int rc = ensure_smem_attribute(reinterpret_cast<const void*>(kv_int4_tiles_kernel<D, T, ALT>), Cfg<D>::kSmem,
                                 &configured, "kv_attention shared memory");
  if (rc != LDB_OK) return rc;
  rc = launch_kernel(kv_int4_tiles_kernel<D, T, ALT>, dim3(p.row_blocks * p.splits, p.c.kv_heads, p.c.batch),
                     dim3(kThreads), Cfg<D>::kSmem, stream, "kv_attention tiles launch", p, status);
  if (rc != LDB_OK || (!ALT && p.splits == 1)) return rc;
  const long long rows = static_cast<long long>(p.c.batch) * p.c.kv_heads * p.rows;
  if (ALT) p.splits *= 2;  // (parts)
  return launch_kernel(kv_tiles_merge_kernel<D, T>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, stream,
                       "kv_attention tiles merge launch", p);
}

template <typename T, bool ALT>
int launch_dim(cudaStream_t stream, const KvTileParams& p, int head_dim, unsigned int* status) {
  if (head_dim == 32) return launch<32, T, ALT>(stream, p, status);
  if (head_dim == 64) return launch<64, T, ALT>(stream, p, status);
  return launch<128, T, ALT>(stream, p, status);
}

// How the tokens are cut: ranges, and parts that they leave.
struct Cuts {
  int ranges, parts;
  bool alternate;
};

// One tile of rows alternates where its ranges are long: it stages its queries twice and leaves two parts a range, but two
// blocks are on their way.  8 key/value heads of 128, 64 rows, us alternating and not: 16384 tokens (8 blocks a
// range) 33 and 31, 32768 (14) 45 and 47, 131072 (57) 109 and 133; 16 items of up to 4096 tokens (32) 65 and 73, of up to
// 16384 (128) 208 and 268; of 64 channels 26 and 24, 36 and 36, 89 and 102, 53 and 56, 174 and 204.
Cuts cuts_of(int batch, int kv_heads, long long rows, int head_dim, long long capacity) {
  const int ranges = kv_tile_splits(batch, kv_heads, rows, head_dim, capacity);
  if (rows > kM || capacity < 25ll * kN * ranges) return {ranges, ranges, false};
  // (twice the parts, in half the time of as many blocks)
  const int pairs = kv_tile_splits(batch, kv_heads, rows, 2 * head_dim, (capacity + 1) / 2);
  return {pairs, 2 * pairs, true};
}

}  // namespace

size_t kv_int4_tile_workspace(int batch, int kv_heads, long long rows, int head_dim, long long capacity) {
  const long long parts = cuts_of(batch, kv_heads, rows, head_dim, capacity).parts;
  return parts <= 1 ? 0 : static_cast<size_t>(parts) * batch * kv_heads * rows * (head_dim + 2) * sizeof(float);
}

int kv_int4_attention_tiles(cudaStream_t stream, KvTileParams p, int head_dim, int dtype, float scale, void* workspace,
                            unsigned int* status) {
  const Cuts cuts = cuts_of(p.c.batch, p.c.kv_heads, p.rows, head_dim, static_cast<long long>(p.c.width) * p.c.page);
  p.row_blocks = (p.rows + 2 * kM - 1) / (2 * kM);
  p.splits = cuts.ranges;
  p.negate = scale < 0.f;
  p.scale_log2 = (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  p.o_part = static_cast<float*>(workspace);
  p.ml_part = p.o_part + static_cast<size_t>(cuts.parts) * p.c.batch * p.c.kv_heads * p.rows * head_dim;
  if (static_cast<long long>(p.row_blocks) * p.splits > 0x7FFFFFFFll || p.c.kv_heads > 65535 || p.c.batch > 65535)
    return fail(LDB_ERR_SHAPE, "kv_attention: %d row blocks, %d heads, %d items", p.row_blocks, p.c.kv_heads,
                p.c.batch);
  if (cuts.alternate)
    return dtype == LDB_F16 ? launch_dim<__half, true>(stream, p, head_dim, status)
                            : launch_dim<__nv_bfloat16, true>(stream, p, head_dim, status);
  return dtype == LDB_F16 ? launch_dim<__half, false>(stream, p, head_dim, status)
                          : launch_dim<__nv_bfloat16, false>(stream, p, head_dim, status);
}

}  // namespace ldb
