// Each head's queries and keys normed and rotated by their token's positions.
//
//   y = x rsqrt(mean(x^2) + eps) gamma                    over a head's D channels
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t)      for pair i of the first 2 P channels
//   t = 2 pi frac(position[axis_i] turns_i)
//
// The pairs are channels (i, i + P), or (2i, 2i + 1) interleaved.  An angle in FP32
// loses its meaning at far positions (2^-24 of 131072 is 0.008); here turns_i is a
// 64-bit fraction of a turn, so position times turns_i modulo 2^64 is exact integer
// arithmetic, and its upper 32 bits are the angle to 2^-32 of a turn at any position.
//
// A warp takes a token, or a few with few heads: the P sines and cosines of each are
// computed once, a pair per lane, and kept in shared memory for all heads.
// Eight channels per lane, as many heads at a time as fit; what a channel becomes is
// f (x own + other times) with its head's norm f, so that sine, cosine and gamma are
// two factors for all heads.
//
// Bound: HBM, each value read and written once; for few tokens the launch.  One B200: 4 x 4097
// tokens of 32 + 8 heads of 128 bf16 66 us (5.1 TB/s; issue 63 %, DRAM 56 %, warps wait for their own values most: four
// rounds are asked for when those before are done), 6400 tokens of 4 + 4 heads of 64 7 us (the chain
// of dependent reads, sines and values), one token of 32 items 3.9 us.

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "fp8.cuh"
#include "packed.cuh"

namespace ldb {
namespace {

struct RopeParams {
  const void* src[2];  // queries, keys
  void* out[2];
  const float* gamma[2];  // [D], null: ones
  long long src_ld[2], src_batch[2], out_ld[2], out_batch[2];
  const unsigned long long* turns;  // [pairs]
  const int* axis;                  // [pairs]
  const int* positions;             // [batch][tokens][axes]
  long long pos_batch, pos_ld;
  int heads[2];
  int tokens, dim, pairs, axes, interleaved, norm, vec;
  int rounds[2], per_warp[2];  // of heads of a token, of a warp: as many heads as fit at a time
  unsigned splits;             // warps of a token
  int token_shift;            // tokens of a warp, as a power of two
  unsigned pairs_inverse;     // 2^16 / pairs, rounded up
  unsigned warps, rows;
  float eps, inv_dim;
};

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxPairs = 128;
// Rounds of values on their way at a time (4 x 4097 tokens of 40 heads of 128: one 92 us, two 72, four 66, six 76).
constexpr int kAhead = 4;

// Eight channels of a row as they are in memory.
template <typename T>
struct Raw {
  static constexpr int kWords = 2 * sizeof(T);
  uint32_t w[kWords];
  // channels 2k and 2k + 1
  __device__ __forceinline__ uint64_t pair(int k) const {
    if constexpr (sizeof(T) == 4) {
      return pack2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return pack2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      return pack2(f.x, f.y);
    }
  }
};

// LANES per head, of eight channels each (the last ones idle where D is not 8 LANES).
template <typename T, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeParams p, unsigned int* status) {
  __shared__ __align__(16) float2 s_turn[kWarps][kMaxPairs];  // (cos, sin)
  pdl_begin();
  const int lane = lane_id();
  const unsigned w = blockIdx.x * kWarps + warp_id();
  if (w >= p.warps) return;
  constexpr int kHeads = 32 / LANES;  // at a time, at_once of each of the warp's tokens
  const int sub = lane / LANES, c0 = (lane % LANES) * 8;
  const unsigned row0 = w / p.splits << p.token_shift;  // the warp's first token
  const int split = static_cast<int>(w % p.splits);
  const int at_once = kHeads >> p.token_shift, mine = sub & (at_once - 1), nth = sub / at_once;
  const unsigned row = min(row0 + nth, p.rows - 1);
  const long long b = row / static_cast<unsigned>(p.tokens);
  const long long token = row - static_cast<unsigned>(b) * p.tokens;
  const bool live = c0 < p.dim && row0 + nth < p.rows;
  const int turned_to = 2 * p.pairs - c0;  // the lane's channels below this one turn (all or none, in halves)
  const bool upper = !INTERLEAVED && c0 >= p.pairs;
  const int away = INTERLEAVED || turned_to <= 0 ? 0 : (upper ? -p.pairs : p.pairs);  // of the other members of its pairs
  const int partner = lane + away / 8;
  float2* turn = s_turn[warp_id()];
  const long long at = b * p.pos_batch + token * p.pos_ld;  // of the lane's token's positions
  const int all = p.pairs << p.token_shift;
  for (int n0 = 0; n0 < all; n0 += 32) {
    const int n = min(n0 + lane, all - 1);
    const int of = static_cast<int>(n * p.pairs_inverse >> 16), i = n - of * p.pairs;  // n / pairs
    const int* position = p.positions + __shfl_sync(0xffffffffu, at, of * at_once * LANES);
    int axis = p.axis[i];
    if (axis < 0 || axis >= p.axes) {
      set_bad_shape(status);
      axis = 0;
    }
    const unsigned long long phase = p.turns[i] * static_cast<unsigned long long>(static_cast<long long>(position[axis]));
    float2 cs;
    sincospif(static_cast<float>(static_cast<int>(phase >> 32)) * 0x1p-31f, &cs.y, &cs.x);
    turn[n] = cs;
  }
  turn += nth * p.pairs;
  __syncwarp();

#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int to = min(p.rounds[which], (split + 1) * p.per_warp[which]);
    int r = split * p.per_warp[which];
    if (r >= to) continue;
    // A token's channel becomes f (x own + other times), f its head's norm: sines, cosines and gamma in two factors.
    uint64_t own[4], times[4];
    {
      float g[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, mate[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
      if (p.gamma[which] && live) {
        load8<float>(p.gamma[which] + c0, g);
        load8<float>(p.gamma[which] + c0 + away, mate);
      }
      // the lane's turns, from the first of its pairs
      const float2* t = turn + (INTERLEAVED ? c0 / 2 : (upper ? c0 - p.pairs : c0));
      const float2 none = make_float2(1.f, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (INTERLEAVED) {
          const float2 cs = 2 * k < turned_to ? t[k] : none;
          own[k] = pack2(cs.x * g[2 * k], cs.x * g[2 * k + 1]);
          times[k] = pack2(-cs.y * g[2 * k + 1], cs.y * g[2 * k]);
        } else {
          const float2 c = turned_to > 0 ? t[2 * k] : none, d = turned_to > 0 ? t[2 * k + 1] : none;
          own[k] = pack2(c.x * g[2 * k], d.x * g[2 * k + 1]);
          const float s0 = c.y * mate[2 * k], s1 = d.y * mate[2 * k + 1];
          times[k] = upper ? pack2(s0, s1) : pack2(-s0, -s1);
        }
      }
    }
    const T* src = static_cast<const T*>(p.src[which]) + b * p.src_batch[which] + token * p.src_ld[which] + c0;
    T* out = static_cast<T*>(p.out[which]) + b * p.out_batch[which] + token * p.out_ld[which] + c0;
    const int heads = live ? p.heads[which] : 0;
    auto load = [&](int head, Raw<T>& raw) {
#pragma unroll
      for (int k = 0; k < Raw<T>::kWords; ++k) raw.w[k] = 0;
      if (head >= heads) return;
      const T* x = src + head * p.dim;
      if (p.vec) {
#pragma unroll
        for (int k = 0; k < Raw<T>::kWords; k += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(x + 4 * k / static_cast<int>(sizeof(T)));
          raw.w[k] = v.x, raw.w[k + 1] = v.y, raw.w[k + 2] = v.z, raw.w[k + 3] = v.w;
        }
      } else {
        __align__(16) T t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = x[j];
#pragma unroll
        for (int k = 0; k < Raw<T>::kWords; ++k) raw.w[k] = reinterpret_cast<const uint32_t*>(t)[k];
      }
    };
    auto finish = [&](int head, const Raw<T>& x) {
      Raw<T> far;  // the other members (nothing where a channel does not turn: an infinity times zero would reach it)
#pragma unroll
      for (int k = 0; k < Raw<T>::kWords; ++k) {
        uint32_t v;
        if (!INTERLEAVED) {
          v = __shfl_sync(0xffffffffu, x.w[k], partner);
        } else {
          v = sizeof(T) == 4 ? x.w[k ^ 1] : __byte_perm(x.w[k], 0, 0x1032);
        }
        far.w[k] = 4 * k / static_cast<int>(sizeof(T)) < turned_to ? v : 0u;
      }
      uint64_t f2 = pack2(1.f, 1.f);
      if (p.norm) {
        uint64_t sums = mul2(x.pair(0), x.pair(0));
#pragma unroll
        for (int k = 1; k < 4; ++k) sums = fma2(x.pair(k), x.pair(k), sums);
        float even, odd;
        unpack2(sums, even, odd);
        float sum = even + odd;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float f = rsqrtf(fmaf(sum, p.inv_dim, p.eps));
        f2 = pack2(f, f);
      }
      float y[8];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        unpack2(mul2(f2, fma2(far.pair(k), times[k], mul2(x.pair(k), own[k]))), y[2 * k], y[2 * k + 1]);
      if (head >= heads) return;
      T* to_row = out + head * p.dim;
      if (p.vec) {
        store8<T>(to_row, y);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) to_row[j] = from_f32<T>(y[j]);
      }
    };
    for (; r < to; r += kAhead) {
      Raw<T> raw[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) load(r + n < to ? (r + n) * at_once + mine : 0x7FFFFFFF, raw[n]);
#pragma unroll
      for (int n = 0; n < kAhead; ++n)
        if (r + n < to) finish((r + n) * at_once + mine, raw[n]);
    }
  }
}

template <typename T>
int launch_rope(cudaStream_t stream, RopeParams& p, long long rows, unsigned int* status) {
  const int lanes = p.dim <= 16 ? 2 : (p.dim <= 32 ? 4 : (p.dim <= 64 ? 8 : (p.dim <= 128 ? 16 : 32)));
  if (rows > 0x7FFFFF00ll) return fail(LDB_ERR_SHAPE, "qk_norm_rope: %lld tokens", rows);
  const long long resident = 32ll * sm_count();
  // Tokens of a warp: as many as its lanes have room for (few heads of few channels leave most idle) while
  // there are tokens enough (183414 tokens of 3 + 3 heads of 32: one a warp 168 us, two 39).
  auto rounds_of = [&](int shift, int i) { const int n = 32 / lanes >> shift; return (p.heads[i] + n - 1) / n; };
  p.token_shift = 0;
  for (int shift = 1; (32 / lanes >> shift) > 0 && (p.pairs << shift) <= kMaxPairs && (rows >> shift) >= resident; ++shift)
    if (rounds_of(shift, 0) + rounds_of(shift, 1) < (rounds_of(p.token_shift, 0) + rounds_of(p.token_shift, 1))
                                                        << (shift - p.token_shift))
      p.token_shift = shift;
  for (int i = 0; i < 2; ++i) p.rounds[i] = rounds_of(p.token_shift, i);
  const long long groups = (rows + (1 << p.token_shift) - 1) >> p.token_shift;  // of tokens that share a warp
  // A warp per round while all of them are resident at once, else all rounds of a token to share its sines.
  int splits = std::max(p.rounds[0], p.rounds[1]);
  while (splits > 1 && groups * splits > resident) splits = (splits + 1) / 2;
  p.splits = splits;
  for (int i = 0; i < 2; ++i) p.per_warp[i] = (p.rounds[i] + splits - 1) / splits;
  p.rows = static_cast<unsigned>(rows);
  p.pairs_inverse = (65535u + std::max(p.pairs, 1)) / std::max(p.pairs, 1);
  p.warps = static_cast<unsigned>(groups * splits);
  const unsigned blocks = (p.warps + kWarps - 1) / kWarps;
  auto pick = [&](auto interleaved) {
    constexpr bool I = decltype(interleaved)::value;
    return lanes == 2    ? rope_kernel<T, 2, I>
           : lanes == 4  ? rope_kernel<T, 4, I>
           : lanes == 8  ? rope_kernel<T, 8, I>
           : lanes == 16 ? rope_kernel<T, 16, I>
                         : rope_kernel<T, 32, I>;
  };
  auto kernel = p.interleaved ? pick(std::true_type{}) : pick(std::false_type{});
  return launch_kernel(kernel, dim3(blocks), dim3(kThreads), 0, stream, "qk_norm_rope launch", p,
                       status);
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_qk_norm_rope(cudaStream_t stream, const ldb_qk_norm_rope_desc* desc) {
  using namespace ldb;
  if (const int rc = check_desc(desc, "qk_norm_rope")) return rc;
  const auto& [struct_size, dtype, q, k, q_out, k_out, q_ld, q_batch, k_ld, k_batch, qo_ld, qo_batch, ko_ld, ko_batch,
               q_gamma, k_gamma, turns, axis, positions, positions_ld, positions_batch, batch, tokens, heads, kv_heads,
               head_dim, pairs, axes, interleaved, norm, eps] = *desc;
  if (batch < 0 || tokens < 0 || heads < 0 || kv_heads < 0)
    return fail(LDB_ERR_SHAPE, "qk_norm_rope: %d items of %d tokens, %d and %d heads", batch, tokens, heads, kv_heads);
  if (dtype != LDB_F16 && dtype != LDB_F32 && dtype != LDB_BF16)
    return fail(LDB_ERR_INVALID, "qk_norm_rope: unknown element type %d", dtype);
  if (head_dim < 16 || head_dim > 256 || head_dim % 16)
    return fail(LDB_ERR_SHAPE, "qk_norm_rope: head_dim %d (a multiple of 16 up to 256)", head_dim);
  if (pairs < 0 || 2 * pairs > head_dim || (!interleaved && pairs % 8) || (pairs > 0 && axes <= 0))
    return fail(LDB_ERR_SHAPE, "qk_norm_rope: %d pairs of %d channels along %d axes (in halves a multiple of 8)", pairs,
                head_dim, axes);
  if (batch == 0 || tokens == 0 || heads + kv_heads == 0) return LDB_OK;
  if ((heads && (!q || !q_out)) || (kv_heads && (!k || !k_out)) || (pairs && (!turns || !axis || !positions)))
    return fail(LDB_ERR_INVALID, "qk_norm_rope: null pointer");
  const long long q_row = static_cast<long long>(heads) * head_dim, k_row = static_cast<long long>(kv_heads) * head_dim;
  if ((tokens > 1 && (q_ld < q_row || k_ld < k_row || qo_ld < q_row || ko_ld < k_row)) ||
      (batch > 1 && (qo_batch < q_row || ko_batch < k_row)))
    return fail(LDB_ERR_SHAPE, "qk_norm_rope: a row stride, or an output's item stride, is below its row");
  for (const float* g : {q_gamma, k_gamma})
    if (reinterpret_cast<uintptr_t>(g) % 16) return fail(LDB_ERR_ALIGNMENT, "qk_norm_rope: gamma must be 16-byte aligned");
  unsigned int* status = device_status_ptr();
  if (!status) return fail(LDB_ERR_CUDA, "qk_norm_rope: no device status word");
  RopeParams p{};
  p.src[0] = q, p.src[1] = k, p.out[0] = q_out, p.out[1] = k_out, p.gamma[0] = q_gamma, p.gamma[1] = k_gamma;
  p.src_ld[0] = q_ld, p.src_ld[1] = k_ld, p.src_batch[0] = q_batch, p.src_batch[1] = k_batch;
  p.out_ld[0] = qo_ld, p.out_ld[1] = ko_ld, p.out_batch[0] = qo_batch, p.out_batch[1] = ko_batch;
  p.turns = turns, p.axis = axis, p.positions = positions, p.pos_batch = positions_batch, p.pos_ld = positions_ld;
  p.heads[0] = heads, p.heads[1] = kv_heads;
  p.tokens = tokens, p.dim = head_dim, p.pairs = pairs, p.axes = axes, p.interleaved = interleaved != 0;
  p.norm = norm != 0, p.eps = eps, p.inv_dim = 1.f / static_cast<float>(head_dim);
  const int es = dtype == LDB_F32 ? 4 : 2;
  p.vec = 1;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    if (reinterpret_cast<uintptr_t>(p.src[i]) % 16 || p.src_ld[i] * es % 16 || p.src_batch[i] * es % 16) p.vec = 0;
    if (reinterpret_cast<uintptr_t>(p.out[i]) % 16 || p.out_ld[i] * es % 16 || p.out_batch[i] * es % 16) p.vec = 0;
  }
  const long long rows = static_cast<long long>(batch) * tokens;
  if (dtype == LDB_F16) return launch_rope<__half>(stream, p, rows, status);
  if (dtype == LDB_BF16) return launch_rope<__nv_bfloat16>(stream, p, rows, status);
  return launch_rope<float>(stream, p, rows, status);
}

}  // extern "C"
