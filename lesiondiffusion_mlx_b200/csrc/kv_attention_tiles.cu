// Attention of many query rows over the paged 8-bit key/value cache, on the
// tcgen05 tensor cores (few rows: kv_attention.cu, whose formulas these are).
//
// One CTA owns two 128-row tiles of one (item, key/value head) and streams
// blocks of 128 tokens once for both; a row is a (query, head of the group) pair.  Scores
// run on the codes as they lie in the cache (kind::f8f6f4): a query row is
// scaled by a power of two and written as e4m3 parts whose products add up in
// the accumulator, two parts for bf16, three for f16, exact but for channels
// 2^-10 (2^-7) below the row's largest, whose error is 2^-18 of that.  The weights
// are f16 in TMEM, so the values become f16 (exact) in shared memory on the
// way: an 8-bit product would need three parts of every weight (2^-11 of each
// is wanted), split by the softmax warps, which are the busiest as it is.  They are 2^7 at
// the row's reference, which may lag 2^8 behind its maximum, so that they use f16's
// range up to 2^15: 11 bits down to 2^-21 of the reference, nothing below 2^-32.
// (A lag of 2^4 leaves room for 2^4 more, but the prompts below with queries four times as
// large, a score's spread of 2^5.8, took 551 us instead of 510.)
//
// Warps: 0 loads code pages (TMA) and page scales, 1 issues the products, 2-3
// turn values into f16, 4-7 and 8-11 run the online softmax of tile 0 and 1,
// one row per thread.  While one tile's scores become weights, the tensor core
// works on the other's.  The output is rescaled in TMEM only when a row's
// reference has to grow by more than 2^8.  Grids that leave SMs idle cut the
// tokens into ranges, merged by a second kernel.
//
// Bound: 4 D flops and one exponential per score; at D = 128 the tensor core
// (1024 cycles per 128 x 128 tile) and the exponentials (1024 cycles) ask for
// as much.  One B200: 4 prompts of 2048 tokens over up to 8000, 32 heads of 128
// over 8, bf16, 483 us (759 TFLOP/s); 6400 f16 tokens over 77, 4 heads of 64,
// 9.9 us.  A block of two tiles takes 4700 cycles: 2000 from a tile's weights to
// its next scores (718 for the value product, 977 for the scores, whose operands
// take 128 bytes a cycle of shared memory), 420 for the maximum, 340 for the
// reference, 1600 for the weights.  Slower: four softmax warpgroups with half a row
// a thread (626 us where two took 527), scores read from TMEM twice (581), and the
// first 64 of the next scores before the value product, in the half of the scores'
// columns that the weights leave free (742 where this took 480: products of half
// the width read the queries twice).

#include <algorithm>

#include "host_common.h"
#include "kv_attention.cuh"

namespace ldb {
namespace {

constexpr int kThreads = 384;
constexpr int kRegsWg0 = 72;      // producer, products, conversion
constexpr int kRegsSoftmax = 216; // a row's 128 scores
static_assert(128 * kRegsWg0 + 256 * kRegsSoftmax <= kThreads * 168, "register split");
constexpr int kM = 128;      // rows per tile
constexpr int kN = 128;      // tokens per block
constexpr int kMeta = 4;     // ring of page factors
constexpr int kGroups = 8;   // of 16 tokens, each of one page (pages under 64 tokens; else the groups come in fours)
constexpr float kFloor = -1.0e30f;  // reference of a row that has seen nothing
constexpr float kGrow = 8.f;        // a reference follows its row's maximum once that is 2^8 above
constexpr int kHeadroom = 7;        // weights are 2^7 at the reference, 2^15 at most; the sum is kept without it

template <int D, int PARTS>
struct Cfg {
  static constexpr uint32_t kLayout = D == 128 ? kSwizzle128 : (D == 64 ? kSwizzle64 : kSwizzle32);
  static constexpr int kPartBytes = kM * D;  // one part of a query tile
  static constexpr int kRawBytes = kN * D;   // codes of a block of K or V
  static constexpr int kSubD = D == 32 ? 32 : 64;  // channels of one f16 value tile
  static constexpr int kSubRow = kSubD * 2;
  static constexpr uint32_t kVLayout = kSubD == 64 ? kSwizzle128 : kSwizzle64;
  static constexpr int kV16Bytes = kN * D * 2;
  static constexpr int kStages = 2;
  static constexpr int kOffK = 2 * PARTS * kPartBytes;
  static constexpr int kOffV = kOffK + kStages * kRawBytes;
  static constexpr int kOffV16 = kOffV + kStages * kRawBytes;
  static constexpr int kOffMeta = kOffV16 + 2 * kV16Bytes;  // [kMeta][8] (see the page warp)
  static constexpr int kOffBad = kOffMeta + kMeta * kGroups * 16;  // NaN met among values that not every row sees
  static constexpr int kOffBar = kOffBad + 16;
  static constexpr int kSmem = 1024 + kOffBar + 256;
  // TMEM: S_t at 128 t, O_t at 256 + 128 t.  D = 128: the weights overwrite
  // their scores; narrower heads have room for them behind O_t, so that the next block's
  // scores need not wait for the value product.
  static constexpr bool kSeparateP = D <= 64;
  static_assert(kSmem <= 232448, "shared memory");
};

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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
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

// FINE: pages under 64 tokens, whose factors change every 16 columns of a
// block; otherwise every 64.  (Fetching them every 16 columns for all pages
// made the softmax, which bounds the kernel, a third longer.)
template <int D, typename T, bool FINE>
__global__ void __launch_bounds__(kThreads, 1)
    kv_tiles_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const KvTileParams p, unsigned int* status) {
  constexpr int PARTS = std::is_same<T, __half>::value ? 3 : 2;
  using C = Cfg<D, PARTS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float4* s_meta = reinterpret_cast<float4*>(smem + C::kOffMeta);
  uint32_t* s_bad = reinterpret_cast<uint32_t*>(smem + C::kOffBad);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;                 // the query parts are written
  uint64_t* k_full = q_full + 1;           // [2] key codes have landed
  uint64_t* k_empty = k_full + 2;          // [2] both tiles' scores have read them
  uint64_t* v_full = k_empty + 2;          // [2] value codes have landed
  uint64_t* v_empty = v_full + 2;          // [2] they have been converted
  uint64_t* v16_full = v_empty + 2;        // [2] f16 values are written
  uint64_t* v16_empty = v16_full + 2;      // [2] the value products have read them
  uint64_t* meta_full = v16_empty + 2;     // [4] page factors are written
  uint64_t* s_full = meta_full + kMeta;    // [2] per tile
  uint64_t* s_free = s_full + 2;           // [2] scores are in registers
  uint64_t* p_ready = s_free + 2;          // [2] weights are in TMEM
  uint64_t* pv_done = p_ready + 2;         // [2]
  uint64_t* drain = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((1 + 12 + kMeta + 8 + 1) * 8 + 8 <= 256, "barrier block");

  const int warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    mbar_init(drain, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 2);
      mbar_init(&v16_full[s], 64);
      mbar_init(&v16_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 4);
      mbar_init(&p_ready[s], 4);
      mbar_init(&pv_done[s], 1);
    }
    for (int s = 0; s < kMeta; ++s) mbar_init(&meta_full[s], 1);
    mbar_init(q_full, p.rows - (p.row_blocks - 1 - static_cast<int>(blockIdx.x) / p.splits) * 2 * kM > kM ? 8 : 4);
    *abort_flag = 0;
    *s_bad = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
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

  if (warp < 4) {
    regs_dec<kRegsWg0>();
    if (warp == 0) {
      // ------------------------------------------------------------ pages
      const int shift = 31 - __clz(p.c.page);
      const int box = min(p.c.page, kN), loads = kN / box;  // pages of a block (one where it is a page)
      const int used = (sp.len + p.c.page - 1) >> shift;
      int batch0 = -32, id = -1;
      float kf = 1.f, ev = 0.f, ev_top = -INFINITY;  // (largest value exponent met)
      bool ok = true;
      int k_loads = 0, v_loads = 0;
      for (int j = 0; ok && j < sp.nblocks; ++j) {
        const int first = ((sp.jb0 + j) * kN) >> shift;
        if (first - batch0 > 32 - loads) {
          batch0 = first;
          const int at = batch0 + lane;
          id = at < used ? p.c.table[sp.b * p.c.table_ld + at] : -1;
          if (at < used && (id < 0 || id >= p.c.pages)) {
            set_bad_shape(status);
            id = -1;
          }
          kf = p.scale_log2;
          ev = -INFINITY;  // (tokens of no page weigh nothing)
          if (id >= 0) {
            const long long unit = static_cast<long long>(id) * p.c.kv_heads + sp.head;
            kf = fp8_pow2(p.c.k_scale[unit] - 127) * p.scale_log2;
            ev = static_cast<float>(p.c.v_scale[unit] - 127);
          }
        }
        const int off = first - batch0;
        const int my_id = __shfl_sync(0xffffffffu, id, (off + lane) & 31);
        const int st = j & 1, ms = j % kMeta;
        const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u;
        ok = warp_wait(&k_empty[st], ph ^ 1u, abort_flag, status);
        if (!ok) break;
        const bool load = lane < loads && my_id >= 0;
        // pages that the table should name and does not: zeros in their place
        const uint32_t holes = __ballot_sync(0xffffffffu, lane < loads && my_id < 0 && first + lane < used);
        auto blank = [&](uint8_t* codes) {
          for (uint32_t rest = holes; rest; rest &= rest - 1) {
            uint4* at = reinterpret_cast<uint4*>(codes + (__ffs(rest) - 1) * box * D);
            for (int i = lane; i < box * D / 16; i += 32) at[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        };
        if (holes) blank(smem + C::kOffK + st * C::kRawBytes);
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, load)) * box * D;
        const int row = (my_id * p.c.kv_heads + sp.head) * p.c.page;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&k_full[st], bytes);
        __syncwarp();
        if (load) tma_load_2d(smem + C::kOffK + st * C::kRawBytes + lane * box * D, &kmap, &k_full[st], 0, row);
        ++k_loads;
        // Factors of the block's eight groups of 16 tokens, once the loads are on their way (slot ms: the
        // scores of block j - 2 are done, so the softmax of block j - 4 is): of the keys, the value
        // scale's exponent, what takes that out of a weight again, and a bit for each group far below the others.
        const int of_group = off + ((lane & 7) * 16 >> shift);
        const float gk = __shfl_sync(0xffffffffu, kf, of_group & 31);
        const float ge = __shfl_sync(0xffffffffu, ev, of_group & 31);
        ev_top = fmaxf(ev_top, ge);
#pragma unroll
        for (int o = 1; o < kGroups; o <<= 1) ev_top = fmaxf(ev_top, __shfl_xor_sync(0xffffffffu, ev_top, o));
        const bool far = kv_far_below(ge, ev_top);
        const uint32_t all_far = __ballot_sync(0xffffffffu, far && lane < kGroups);
        if (lane < kGroups)
          s_meta[ms * kGroups + lane] =
              make_float4(gk, ge, far ? 0.f : fp8_pow2(-max(static_cast<int>(ge), -127) - kHeadroom),
                          __uint_as_float(all_far));
        __syncwarp();
        if (lane == 0) mbar_arrive(&meta_full[ms]);
        ok = warp_wait(&v_empty[st], ph ^ 1u, abort_flag, status);
        if (!ok) break;
        if (holes) blank(smem + C::kOffV + st * C::kRawBytes);
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&v_full[st], bytes);
        __syncwarp();
        if (load) tma_load_2d(smem + C::kOffV + st * C::kRawBytes + lane * box * D, &vmap, &v_full[st], 0, row);
        ++v_loads;
      }
      if (*abort_flag) {
        // Let the loads in flight land before the CTA gives up its shared memory.
        volatile int never = 0;
        for (int n = max(0, k_loads - 2); n < k_loads; ++n)
          mbar_wait(&k_full[n & 1], static_cast<uint32_t>(n >> 1) & 1u, &never, status);
        for (int n = max(0, v_loads - 2); n < v_loads; ++n)
          mbar_wait(&v_full[n & 1], static_cast<uint32_t>(n >> 1) & 1u, &never, status);
      }
    } else if (warp == 1) {
      // --------------------------------------------------------- products
      if (sp.nblocks > 0) {
        constexpr uint32_t idesc_qk = (1u << 4) | (kN >> 3 << 17) | (kM >> 4 << 24);  // e4m3 x e4m3 -> f32
        constexpr uint32_t idesc_pv = make_idesc_f16(kM, D, 0u, 0u, 1u);
        auto scores = [&](int t, int j) {
          const uint32_t k_addr = smem_u32(smem + C::kOffK + (j & 1) * C::kRawBytes);
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            const uint32_t q_addr = smem_u32(smem + (t * PARTS + part) * C::kPartBytes);
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
              umma_ss_f8(tmem + t * 128, make_smem_desc(q_addr + k * 32, 16, 8 * D, C::kLayout),
                         make_smem_desc(k_addr + k * 32, 16, 8 * D, C::kLayout), idesc_qk,
                         (part > 0 || k > 0) ? 1u : 0u);
          }
          umma_commit_warp(&s_full[t]);
        };
        auto values = [&](int t, int j) {
          const uint32_t v_addr = smem_u32(smem + C::kOffV16 + (j & 1) * C::kV16Bytes);
          const uint32_t p_tmem = C::kSeparateP ? tmem + 256 + t * 128 + 64 : tmem + t * 128;
#pragma unroll
          for (int k = 0; k < kN / 16; ++k)  // (value tiles of 64 channels lie kN rows apart)
            umma_ts_warp(tmem + 256 + t * 128, p_tmem + k * 8,
                         make_smem_desc(v_addr + k * 16 * C::kSubRow, kN * C::kSubRow, 8 * C::kSubRow, C::kVLayout),
                         idesc_pv, (j > 0 || k > 0) ? 1u : 0u);
          umma_commit_warp(&pv_done[t]);
        };
        bool ok = warp_wait(q_full, 0, abort_flag, status);
        for (int j = 0; ok && j <= sp.nblocks; ++j) {
          const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u, was = static_cast<uint32_t>(j - 1) & 1u;
          if (j < sp.nblocks) ok = warp_wait(&k_full[j & 1], ph, abort_flag, status);
          if (ok && j > 0)
            ok = warp_wait(&v16_full[(j - 1) & 1], static_cast<uint32_t>((j - 1) >> 1) & 1u, abort_flag, status);
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
          if (ok && j > 0) umma_commit_warp(&v16_empty[(j - 1) & 1]);
        }
        umma_commit_warp(drain);
        volatile int never = 0;
        mbar_wait(drain, 0, &never, status);
      }
    } else {
      // -------------------------------------------------- values to f16
      const int tid = threadIdx.x - 64;
      constexpr int kUnits = D / 16;      // 16-byte units of a token
      constexpr int kStep = 64 / kUnits;  // tokens of a round (a multiple of eight: one swizzle pattern for all rounds)
      // 16 channels are two units of a f16 row; lanes of the second value tile
      // write theirs in the other order (the same banks otherwise).
      const int tok0 = tid / kUnits, chunk = tid % kUnits, sub = chunk * 16 / C::kSubD;
      const bool swap = sub & 1;
      const int at_raw = swizzle_offset(tid * 16, D);
      const int at_out = tok0 * C::kSubRow + (chunk * 32) % C::kSubRow;
      const int at_first = sub * kN * C::kSubRow + swizzle_offset(at_out + (swap ? 16 : 0), C::kSubRow);
      const int at_second = sub * kN * C::kSubRow + swizzle_offset(at_out + (swap ? 0 : 16), C::kSubRow);
      bool ok = true;
      for (int j = 0; ok && j < sp.nblocks; ++j) {
        const int st = j & 1;
        const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u;
        ok = warp_wait(&v_full[st], ph, abort_flag, status) &&
             warp_wait(&v16_empty[st], ph ^ 1u, abort_flag, status);
        if (!ok) break;
        const uint8_t* raw = smem + C::kOffV + st * C::kRawBytes;
        uint8_t* out = smem + C::kOffV16 + st * C::kV16Bytes;
        const int j0 = (sp.jb0 + j) * kN;
        // unit tid + 64 n: the same channels of every kStep-th token
        auto convert = [&](int n, uint4 w, auto masked) {
          if constexpr (decltype(masked)::value) {
            // Where some rows may not see a token its NaN becomes zero here, and
            // the rows that do see it get the NaN at the end.
            if (j0 + tok0 + n * kStep >= sp.len) w = make_uint4(0, 0, 0, 0);
            if (kv_nan_codes(w.x) | kv_nan_codes(w.y) | kv_nan_codes(w.z) | kv_nan_codes(w.w)) {
              *s_bad = 1;
              w = make_uint4(kv_without_nan(w.x), kv_without_nan(w.y), kv_without_nan(w.z), kv_without_nan(w.w));
            }
          }
          const uint4 lo =
              make_uint4(fp8_unpack2(w.x), fp8_unpack2(w.x >> 16), fp8_unpack2(w.y), fp8_unpack2(w.y >> 16));
          const uint4 hi =
              make_uint4(fp8_unpack2(w.z), fp8_unpack2(w.z >> 16), fp8_unpack2(w.w), fp8_unpack2(w.w >> 16));
          *reinterpret_cast<uint4*>(out + n * kStep * C::kSubRow + at_first) = swap ? hi : lo;
          *reinterpret_cast<uint4*>(out + n * kStep * C::kSubRow + at_second) = swap ? lo : hi;
        };
        auto block = [&](auto masked) {
#pragma unroll
          for (int n0 = 0; n0 < kN / kStep; n0 += 4) {
            uint4 w[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) w[n] = *reinterpret_cast<const uint4*>(raw + (n0 + n) * kStep * D + at_raw);
#pragma unroll
            for (int n = 0; n < 4; ++n) convert(n0 + n, w[n], masked);
          }
        };
        // (two loops: with the test inside one the prompts of the head comment took 641 us instead of 493)
        if (j0 + kN > sp.open) {
          block(std::true_type{});
        } else {
          block(std::false_type{});
        }
        fence_proxy_async_smem();
        mbar_arrive(&v16_full[st]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_empty[st]);
      }
    }
  } else {
    regs_inc<kRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    const int t = (warp - 4) >> 2;  // tile of this warpgroup
    const int quarter = warp & 3;   // TMEM lanes this warp may access
    const int local = quarter * 32 + lane;
    const int row = sp.row0 + t * kM + local;
    const bool live = row < p.rows;
    const int i = live ? row / p.group : 0, gq = live ? row % p.group : 0;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tmem_s = tmem + t * 128 + lane_base;
    const uint32_t tmem_o = tmem + 256 + t * 128 + lane_base;
    const uint32_t tmem_p = C::kSeparateP ? tmem_o + 64 : tmem_s;
    const int limit = p.causal && live ? min(sp.len, sp.len - p.queries + i + 1) : sp.len;  // keys that the row sees
    float qs = 1.f;
    if (t < sp.tiles && sp.nblocks > 0) {
      // Query rows in parts: the largest magnitude to [128, 256); a NaN stays
      // one, an infinity makes the row's factor one (of a row that sees any key).
      // D / 8 neighbouring lanes read a row, eight channels each: with a row per
      // lane it took 10500 cycles at D = 128 in three parts, now 8400.
      constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // lanes of a row, rows at a time
      const T* src = static_cast<const T*>(p.q) + sp.b * p.q_batch + i * p.q_ld +
                     (static_cast<long long>(sp.head) * p.group + gq) * D;
      const int part_lane = lane % kLanes;
      auto rows_from = [&](int n0, uint4(&raw)[4]) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int from = (n0 + n) * kRows + lane / kLanes;  // row of the warp, and the lane that owns it
          const T* at = reinterpret_cast<const T*>(__shfl_sync(
                            0xffffffffu, reinterpret_cast<unsigned long long>(src), from & 31)) + 8 * part_lane;
          raw[n] = make_uint4(0, 0, 0, 0);
          if (from < 32 && sp.row0 + t * kM + quarter * 32 + from < p.rows) {
            if (p.q_vec) {
              raw[n] = *reinterpret_cast<const uint4*>(at);
            } else {
              const uint16_t* h = reinterpret_cast<const uint16_t*>(at);
              raw[n] = make_uint4(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16,
                                  h[4] | static_cast<uint32_t>(h[5]) << 16, h[6] | static_cast<uint32_t>(h[7]) << 16);
            }
          }
        }
      };
      float top_of = 0.f;  // largest magnitude of the lane's own row
      uint4 next[4];
      rows_from(0, next);
#pragma unroll 1
      for (int n0 = 0; n0 < kLanes; n0 += 4) {
        uint4 raw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) raw[k] = next[k];
        rows_from(n0 + 4, next);
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          const int n = n0 + k4;
          const uint32_t w[4] = {raw[k4].x, raw[k4].y, raw[k4].z, raw[k4].w};
          float m = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 x = kv_unpack2<T>(w[k]);
            m = fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          const float own = __shfl_sync(0xffffffffu, m, (lane % kRows) * kLanes);
          if (lane / kRows == n) top_of = own;
          const float factor = fp8_pow2(7 - kv_query_exponent(m));
          const float inv = p.negate ? -factor : factor;
          uint32_t parts[PARTS][2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = kv_unpack2<T>(w[2 * k]), y = kv_unpack2<T>(w[2 * k + 1]);
            __half2 rest[2] = {__floats2half2_rn(x.x * inv, x.y * inv), __floats2half2_rn(y.x * inv, y.y * inv)};
#pragma unroll
            for (int part = 0; part < PARTS; ++part) parts[part][k] = kv_split_part<1>(rest);
          }
          const int at = swizzle_offset((quarter * 32 + n * kRows + lane / kLanes) * D + 8 * part_lane, D);
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            *reinterpret_cast<uint2*>(smem + (t * PARTS + part) * C::kPartBytes + at) =
                make_uint2(parts[part][0], parts[part][1]);
        }
      }
      qs = fp8_is_finite(top_of) || limit <= 0 ? fp8_pow2(kv_query_exponent(top_of) - 7) : fp8_nan();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    float top = kFloor, l = 0.f;
    bool ok = t < sp.tiles;
    // The blocks from j on; without WITH_FAR, up to the first that has pages far below the others
    // (rare).  Two loops: with those pages' terms in one, wherever they stood, the
    // prompts of the head comment took 494 to 526 us where two take 484.
    auto blocks = [&](int j, auto with_far) {
      constexpr bool WITH_FAR = decltype(with_far)::value;
      for (; ok && j < sp.nblocks; ++j) {
        ok = warp_wait(&s_full[t], static_cast<uint32_t>(j) & 1u, abort_flag, status) &&
             warp_wait(&meta_full[j % kMeta], static_cast<uint32_t>(j / kMeta) & 1u, abort_flag, status);
        if (!ok) break;
        tc_fence_after();
        uint32_t sr[kN];
#pragma unroll
        for (int c0 = 0; c0 < kN; c0 += 32) {
          uint32_t(&chunk)[32] = *reinterpret_cast<uint32_t(*)[32]>(&sr[c0]);
          tmem_ld32(tmem_s + c0, chunk);
        }
        const float4* meta = s_meta + (j % kMeta) * kGroups;
        const uint32_t far = __float_as_uint(meta[0].w);  // groups of 16 tokens
        tmem_wait_ld();
        if (far && !WITH_FAR) break;
        if constexpr (C::kSeparateP) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[t]);
        }
        const int j0 = (sp.jb0 + j) * kN;
        if (j0 + kN > sp.open) {  // hidden keys count nothing
#pragma unroll
          for (int c = 0; c < kN; ++c)
            if (j0 + c >= limit) sr[c] = 0xFF800000u;
        }
        constexpr int kCols = FINE ? 16 : 64;  // columns of one page
        auto factor = [&](float kf) {
          const float f = qs * kf;
          return f < 1.2e-38f ? 1.2e-38f : f;  // (-inf times zero would be a NaN)
        };
        float mx = kFloor;
#pragma unroll
        for (int c0 = 0; c0 < kN; c0 += kCols) {
          // independent chains of 3-input maxima, folded
          float m4[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            m4[k] = fmaxf(__uint_as_float(sr[c0 + 2 * k]), __uint_as_float(sr[c0 + 2 * k + 1]));
#pragma unroll
          for (int c = 8; c < kCols; c += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              m4[k] = max3(m4[k], __uint_as_float(sr[c0 + c + 2 * k]), __uint_as_float(sr[c0 + c + 2 * k + 1]));
          const float4 v = meta[c0 / 16];
          mx = fmaxf(mx, fmaf(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), factor(v.x), v.y));
        }
        const bool first = j == 0;
        const bool grow = first || mx - top > kGrow;
        const float next = grow ? fmaxf(top, mx) : top;
        const float half = first ? 0.f : ex2_approx(0.5f * (top - next)), alpha = half * half;
        if (j > 0) {
          // the value product of the block before is done: its weights' place is free, O is whole
          ok = warp_wait(&pv_done[t], static_cast<uint32_t>(j - 1) & 1u, abort_flag, status);
          if (!ok) break;
          tc_fence_after();
          if (__any_sync(0xffffffffu, grow)) {
            const float scale = grow ? alpha : 1.f;
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += 16) {
              uint32_t r[16];
              tmem_ld16(tmem_o + c0, r);
              tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < 16; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * scale);
              tmem_st16(tmem_o + c0, r);
            }
            tmem_wait_st();
          }
        }
        if (grow) {
          l = kv_scaled(l, half);
          top = next;
        }
        if constexpr (WITH_FAR) {
#pragma unroll
          for (int c0 = 0; c0 < kN; c0 += kCols) {
            if (!((far >> (c0 / 16)) & 1u)) continue;
            const float f = factor(meta[c0 / 16].x);
#pragma unroll
            for (int c = 0; c < kCols; ++c) l += ex2_approx(fmaf(__uint_as_float(sr[c0 + c]), f, -top));
          }
        }
#pragma unroll
        for (int c0 = 0; c0 < kN; c0 += kCols) {
          const float4 v = meta[c0 / 16];
          const float f = factor(v.x);
          const float ref = top - kHeadroom;
          const uint64_t f2 = pack2(f, f), shift = pack2(v.y - ref, v.y - ref);
          uint64_t sum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
          for (int h = 0; h < kCols; h += 16) {
            uint32_t packed[8];
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              const int at = c0 + h + c;
              float x0, x1;
              unpack2(fma2(pack2(__uint_as_float(sr[at]), __uint_as_float(sr[at + 1])), f2, shift), x0, x1);
              const float e0 = ex2_approx(x0), e1 = ex2_approx(x1);
              sum2[(c >> 1) & 1] = add2(sum2[(c >> 1) & 1], pack2(e0, e1));
              const __half2 w = __floats2half2_rn(e0, e1);
              packed[c / 2] = *reinterpret_cast<const uint32_t*>(&w);
            }
            tmem_st8(tmem_p + ((c0 + h) >> 1), packed);
          }
          float a, b;
          unpack2(add2(sum2[0], sum2[1]), a, b);
          l = fmaf(a + b, v.z, l);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);
      }
      return j;
    };
    const int rest = blocks(0, std::false_type{});
    if (ok && rest < sp.nblocks) blocks(rest, std::true_type{});
    if (ok && sp.nblocks > 0)
      ok = warp_wait(&pv_done[t], static_cast<uint32_t>(sp.nblocks - 1) & 1u, abort_flag, status) &&
           warp_wait(&v16_full[(sp.nblocks - 1) & 1], static_cast<uint32_t>((sp.nblocks - 1) >> 1) & 1u, abort_flag,
                     status);  // (done as well: orders the reads of s_bad)
    if (ok) {
      tc_fence_after();
      const int split = blockIdx.x % p.splits;
      const long long part =
          ((static_cast<long long>(split) * p.c.batch + sp.b) * p.c.kv_heads + sp.head) * p.rows + row;
      T* dst = static_cast<T*>(p.out) + sp.b * p.out_batch + i * p.out_ld +
               (static_cast<long long>(sp.head) * p.group + gq) * D;
      const float inv = l == 0.f ? 0.f : fp8_pow2(-kHeadroom) / l;
      // (one range: rows to shared memory, where the queries were, and from there D /
      // 8 lanes a row; stored a row per lane they took 6000 cycles at D = 128, now 4200)
      constexpr int kChunks = D / 8, kSpread = kChunks < 8 ? kChunks - 1 : 7;  // 16-byte pieces of an output row
      uint8_t* rows = smem + t * PARTS * C::kPartBytes + quarter * 32 * D * 2;
      static_assert(PARTS >= 2, "an output tile fits where its queries were");
#pragma unroll 2
      for (int c0 = 0; c0 < D; c0 += 16) {
        uint32_t r[16];
        if (sp.nblocks > 0) {
          tmem_ld16(tmem_o + c0, r);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) r[c] = 0;
        }
        if (p.splits > 1) {
          if (live) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              reinterpret_cast<float4*>(p.o_part + part * D + c0)[c] =
                  make_float4(__uint_as_float(r[4 * c]), __uint_as_float(r[4 * c + 1]), __uint_as_float(r[4 * c + 2]),
                              __uint_as_float(r[4 * c + 3]));
          }
          __syncwarp();  // the next read of TMEM is the whole warp's
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = __uint_as_float(r[8 * h + c]) * inv;
            store8<T>(reinterpret_cast<T*>(rows + lane * D * 2 + ((c0 / 8 + h) ^ (lane & kSpread)) * 16), v);
          }
        }
      }
      if (p.splits == 1) {
        __syncwarp();
        constexpr int kLanes = D / 8, kRows = 32 / kLanes;
#pragma unroll 4
        for (int n = 0; n < kLanes; ++n) {
          const int from = n * kRows + lane / kLanes, chunk = lane % kLanes;
          T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), from)) +
                  8 * chunk;
          if (sp.row0 + t * kM + quarter * 32 + from >= p.rows) continue;
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
      if (p.splits > 1 && live) *reinterpret_cast<float2*>(p.ml_part + part * 2) = make_float2(top, l);
      tc_fence_before();
      if (sp.nblocks > 0 && live && *s_bad != 0) {
        // Rare: NaN among the values of the blocks that `open` cuts, whose product
        // left them out.  Looked up again in the cache, token by token, by each row.
        const int to = min(limit, (sp.jb0 + sp.nblocks) * kN);
        for (int tok = max(sp.jb0, max(sp.open, 0) / kN) * kN; tok < to; ++tok) {
          const int id = p.c.table[sp.b * p.c.table_ld + tok / p.c.page];
          if (id < 0 || id >= p.c.pages) continue;
          const uint8_t* v =
              p.c.v + ((static_cast<long long>(id) * p.c.kv_heads + sp.head) * p.c.page + tok % p.c.page) * D;
          for (int c = 0; c < D; ++c) {
            if ((v[c] & 0x7F) != 0x7F) continue;
            if (p.splits > 1) {
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

// One warp per row: the ranges' parts in order.
template <int D, typename T>
__global__ void __launch_bounds__(256) kv_tiles_merge_kernel(const KvTileParams p) {
  pdl_begin();
  const long long total = static_cast<long long>(p.c.batch) * p.c.kv_heads * p.rows;
  const long long at = blockIdx.x * 8ll + warp_id();
  if (at >= total) return;
  const int lane = lane_id();
  float m = kFloor;
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

template <int D, typename T, bool FINE>
int launch(cudaStream_t stream, const KvTileParams& p, unsigned int* status) {
  using C = Cfg<D, std::is_same<T, __half>::value ? 3 : 2>;
  static unsigned long long configured = 0;
  int rc = ensure_smem_attribute(reinterpret_cast<const void*>(kv_tiles_kernel<D, T, FINE>), C::kSmem, &configured,
                                 "kv_attention shared memory");
  if (rc != LDB_OK) return rc;
  CUtensorMap kmap, vmap;
  const uint64_t dims[2] = {static_cast<uint64_t>(D),
                            static_cast<uint64_t>(p.c.pages) * p.c.kv_heads * p.c.page};
  const uint64_t strides[1] = {static_cast<uint64_t>(D)};
  const uint32_t box[2] = {static_cast<uint32_t>(D), static_cast<uint32_t>(std::min(p.c.page, kN))};
  rc = encode_tiled_u8(&kmap, p.c.k, 2, dims, strides, box, D);
  if (rc == LDB_OK) rc = encode_tiled_u8(&vmap, p.c.v, 2, dims, strides, box, D);
  if (rc != LDB_OK) return rc;
  rc = launch_kernel(kv_tiles_kernel<D, T, FINE>, dim3(p.row_blocks * p.splits, p.c.kv_heads, p.c.batch),
                     dim3(kThreads), C::kSmem, stream, "kv_attention tiles launch", kmap, vmap, p, status);
  if (rc != LDB_OK || p.splits == 1) return rc;
  const long long rows = static_cast<long long>(p.c.batch) * p.c.kv_heads * p.rows;
  return launch_kernel(kv_tiles_merge_kernel<D, T>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, stream,
                       "kv_attention tiles merge launch", p);
}

template <int D, typename T>
int launch_page(cudaStream_t stream, const KvTileParams& p, unsigned int* status) {
  return p.c.page < 64 ? launch<D, T, true>(stream, p, status) : launch<D, T, false>(stream, p, status);
}

template <typename T>
int launch_dim(cudaStream_t stream, const KvTileParams& p, int head_dim, unsigned int* status) {
  if (head_dim == 32) return launch_page<32, T>(stream, p, status);
  if (head_dim == 64) return launch_page<64, T>(stream, p, status);
  return launch_page<128, T>(stream, p, status);
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

size_t kv_tile_workspace(int batch, int kv_heads, long long rows, int head_dim, long long capacity) {
  const long long ctas = (rows + 2 * kM - 1) / (2 * kM) * kv_heads * batch;
  const long long splits = capacity < 0 ? std::min(32ll, 4ll * sm_count() / std::max(1ll, ctas))
                                        : kv_tile_splits(batch, kv_heads, rows, head_dim, capacity);
  return splits <= 1 ? 0 : static_cast<size_t>(splits) * batch * kv_heads * rows * (head_dim + 2) * sizeof(float);
}

int kv_attention_tiles(cudaStream_t stream, KvTileParams p, int head_dim, int dtype, float scale, void* workspace,
                       unsigned int* status) {
  p.row_blocks = (p.rows + 2 * kM - 1) / (2 * kM);
  p.splits = kv_tile_splits(p.c.batch, p.c.kv_heads, p.rows, head_dim, static_cast<long long>(p.c.width) * p.c.page);
  p.negate = scale < 0.f;
  p.scale_log2 = (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  p.o_part = static_cast<float*>(workspace);
  p.ml_part = p.o_part + static_cast<size_t>(p.splits) * p.c.batch * p.c.kv_heads * p.rows * head_dim;
  if (static_cast<long long>(p.row_blocks) * p.splits > 0x7FFFFFFFll || p.c.kv_heads > 65535 || p.c.batch > 65535)
    return fail(LDB_ERR_SHAPE, "kv_attention: %d row blocks, %d heads, %d items", p.row_blocks, p.c.kv_heads,
                p.c.batch);
  return dtype == LDB_F16 ? launch_dim<__half>(stream, p, head_dim, status)
                          : launch_dim<__nv_bfloat16>(stream, p, head_dim, status);
}

}  // namespace ldb
