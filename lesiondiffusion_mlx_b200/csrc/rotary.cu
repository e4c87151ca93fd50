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
// A warp takes a token: its P sines and cosines are computed once, a pair per
// lane, and kept in shared memory for all heads; eight channels per lane, as
// many heads at a time as fit.
//
// Bound: HBM, each value read and written once; for few tokens the launch.

#include "host_common.h"
#include "fp8.cuh"

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
  int rounds, per_warp;  // heads of a token, of a warp, in rounds of as many as fit
  unsigned splits;       // warps of a token
  unsigned warps;
  float eps, inv_dim;
};

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxPairs = 128;

// LANES per head, of eight channels each (the last ones idle where D is not 8 LANES).
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeParams p, unsigned int* status) {
  __shared__ __align__(16) float2 s_turn[kWarps][kMaxPairs];  // (cos, sin)
  pdl_begin();
  const int lane = lane_id();
  const unsigned w = blockIdx.x * kWarps + warp_id();
  if (w >= p.warps) return;
  const unsigned row = w / p.splits;
  const int split = static_cast<int>(w - row * p.splits);
  const long long b = row / static_cast<unsigned>(p.tokens);
  const long long token = row - static_cast<unsigned>(b) * p.tokens;
  float2* turn = s_turn[warp_id()];
  const int* position = p.positions + b * p.pos_batch + token * p.pos_ld;
  for (int i = lane; i < p.pairs; i += 32) {
    int axis = p.axis[i];
    if (axis < 0 || axis >= p.axes) {
      set_bad_shape(status);
      axis = 0;
    }
    const unsigned long long phase = p.turns[i] * static_cast<unsigned long long>(static_cast<long long>(position[axis]));
    float2 cs;
    sincospif(static_cast<float>(static_cast<int>(phase >> 32)) * 0x1p-31f, &cs.y, &cs.x);
    turn[i] = cs;
  }
  __syncwarp();
  constexpr int kHeads = 32 / LANES;  // at a time
  const int sub = lane / LANES, c0 = (lane % LANES) * 8;
  const bool live = c0 < p.dim;
  // the lane's pairs, and which member of them it holds
  const int first = p.interleaved ? c0 / 2 : (c0 < p.pairs ? c0 : c0 - p.pairs);
  const bool turned = c0 < 2 * p.pairs;  // (some of the lane's channels)
  const bool upper = !p.interleaved && c0 >= p.pairs;
  const int partner = lane + (p.interleaved || !turned ? 0 : (upper ? -p.pairs / 8 : p.pairs / 8));
  const int turned_to = min(8, 2 * p.pairs - c0);  // the lane's channels below this one turn
  float cs[8], sn[8];  // by channel
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = p.interleaved ? first + j / 2 : first + j;
    const float2 t = turned && i < p.pairs ? turn[i] : make_float2(0.f, 0.f);
    const bool second = p.interleaved ? (j & 1) : upper;
    cs[j] = t.x;
    sn[j] = second ? t.y : -t.y;
  }
  const int all = p.heads[0] + p.heads[1];
  const int to = min(p.rounds, (split + 1) * p.per_warp);
  for (int r = split * p.per_warp; r < to; ++r) {
    int head = r * kHeads + sub;
    const bool here = live && head < all;
    const int which = head >= p.heads[0] ? 1 : 0;
    if (which) head -= p.heads[0];
    float x[8];
    if (here) {
      const T* src = static_cast<const T*>(p.src[which]) + b * p.src_batch[which] + token * p.src_ld[which] +
                     static_cast<long long>(head) * p.dim + c0;
      if (p.vec) {
        load8<T>(src, x);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = to_f32<T>(src[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
    }
    if (p.norm) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float f = rsqrtf(fmaf(sum, p.inv_dim, p.eps));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= f;
    }
    if (here && p.gamma[which]) {
      float g[8];
      load8<float>(p.gamma[which] + c0, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= g[j];
    }
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float other = p.interleaved ? x[j ^ 1] : __shfl_sync(0xffffffffu, x[j], partner);
      y[j] = j < turned_to ? fmaf(x[j], cs[j], other * sn[j]) : x[j];
    }
    if (here) {
      T* out = static_cast<T*>(p.out[which]) + b * p.out_batch[which] + token * p.out_ld[which] +
               static_cast<long long>(head) * p.dim + c0;
      if (p.vec) {
        store8<T>(out, y);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = from_f32<T>(y[j]);
      }
    }
  }
}

template <typename T>
int launch_rope(cudaStream_t stream, RopeParams& p, long long rows, unsigned int* status) {
  const int lanes = p.dim <= 16 ? 2 : (p.dim <= 32 ? 4 : (p.dim <= 64 ? 8 : (p.dim <= 128 ? 16 : 32)));
  const int at_a_time = 32 / lanes;
  p.rounds = (p.heads[0] + p.heads[1] + at_a_time - 1) / at_a_time;
  // A warp per round while all of them are resident at once, else rounds enough to share the sines.
  const long long resident = 32ll * sm_count();
  p.per_warp = 1;
  while (p.per_warp < p.rounds && p.per_warp < 8 && rows * ((p.rounds + p.per_warp - 1) / p.per_warp) > resident)
    p.per_warp *= 2;
  if (p.per_warp > p.rounds) p.per_warp = p.rounds;
  p.splits = (p.rounds + p.per_warp - 1) / p.per_warp;
  if (rows * p.splits > 0x7FFFFF00ll) return fail(LDB_ERR_SHAPE, "qk_norm_rope: %lld tokens of %d heads", rows, p.heads[0]);
  p.warps = static_cast<unsigned>(rows * p.splits);
  const unsigned blocks = (p.warps + kWarps - 1) / kWarps;
  auto kernel = lanes == 2    ? rope_kernel<T, 2>
                : lanes == 4  ? rope_kernel<T, 4>
                : lanes == 8  ? rope_kernel<T, 8>
                : lanes == 16 ? rope_kernel<T, 16>
                              : rope_kernel<T, 32>;
  return launch_kernel(kernel, dim3(blocks), dim3(kThreads), 0, stream, "qk_norm_rope launch", p,
                       status);
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_qk_norm_rope(cudaStream_t stream, const void* q, long long q_ld, long long q_batch, const void* k,
                     long long k_ld, long long k_batch, int dtype, const float* q_gamma, const float* k_gamma,
                     float eps, int norm, const unsigned long long* turns, const int* axis, int pairs, int axes,
                     int interleaved, const int* positions, long long positions_ld, long long positions_batch,
                     void* q_out, long long qo_ld, long long qo_batch, void* k_out, long long ko_ld, long long ko_batch,
                     int batch, int tokens, int heads, int kv_heads, int head_dim) {
  using namespace ldb;
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
