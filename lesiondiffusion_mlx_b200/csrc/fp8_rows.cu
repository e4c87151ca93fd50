// Row quantization to the 8-bit format of fp8.cuh: the root-mean-square norm
// with the residual's addition, plain rows, and the one-time packing of
// weights.
//
//   h = x + r                                (FP32; stored rounded to x's type)
//   y = h * rsqrt(mean(h^2) + eps) * gamma   (FP32, from the unrounded h)
//   code = e4m3(y * 2^-e), e per row and 128 channels
//
// Bound: HBM.  x and r are read once (2 x 2 bytes a channel in 16 bits), h and
// the codes written once (2 + 1 bytes): the row stays in registers between the
// sum of squares and the rounding, 8 consecutive channels a lane, so that 16
// lanes hold the 128 channels of a scale and find its maximum with four
// shuffles.  Rows of up to 1024 channels take one warp (no barrier), wider rows
// a block; the grid is resident and walks the rows.  One B200: 51201 x 1000 bf16
// with a residual 68 us (5.3 TB/s, 0.82 of the copy rate), 6400 x 256 f16 3.5
// us, one row 2.5 us.

#include <algorithm>

#include "fp8.cuh"
#include "host_common.h"

namespace ldb {
namespace {

struct RowsParams {
  const void* x;
  const void* residual;  // may be null
  const float* gamma;    // may be null (ones)
  void* h;               // may be null
  uint8_t* codes;
  uint8_t* scales;
  long long x_ld, r_ld, h_ld, codes_ld, scales_ld;
  int rows, channels;
  float eps;
};

// A lane's eight channels: consecutive where channels, strides and addresses allow
// 16-byte accesses (VEC), else every 32nd, so that a warp's narrow accesses are
// consecutive (4937 x 6189 bf16 with a residual took 126 us with eight consecutive
// channels a lane, 76 so; 4937 x 6192 takes 49).
template <bool VEC>
__device__ __forceinline__ int channel_of(int warp, int lane, int j) {
  return VEC ? (warp * 32 + lane) * 8 + j : warp * 256 + j * 32 + lane;
}
// Eight channels (zero past the row's end).
template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T* row, int warp, int lane, int channels, float (&v)[8]) {
  if constexpr (VEC) {
    load8<T>(row + channel_of<VEC>(warp, lane, 0), v);
  } else {
    const T* at = row + channel_of<VEC>(warp, lane, 0);
    const int left = channels - channel_of<VEC>(warp, lane, 0);
    if (warp * 256 + 256 <= channels) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(at[32 * j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 32 * j < left ? to_f32<T>(at[32 * j]) : 0.f;
    }
  }
}

__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// Quantize the 128 channels that 16 neighbouring lanes hold, 8 each; every
// lane of the warp takes part, lanes with `live` store.
__device__ __forceinline__ void quantize_block(float (&y)[8], bool live, bool first, uint8_t* codes, uint8_t* scale) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));  // a NaN leaves the maximum as it is
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  // Infinities (rare): out of the maximum, and NaN before the rounding.
  if (__any_sync(0xffffffffu, !fp8_is_finite(amax))) {
    amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (fp8_is_finite(y[j])) {
        amax = fmaxf(amax, fabsf(y[j]));
      } else {
        y[j] = fp8_nan();
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  const int e = fp8_exponent(amax);
  const float inv = fp8_pow2(-e);
  if (live) {
    uint2 packed;
    packed.x = fp8_pack4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
    packed.y = fp8_pack4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
    *reinterpret_cast<uint2*>(codes) = packed;
    if (first) *scale = static_cast<uint8_t>(e + 127);
  }
}

// The same for lanes that hold every 32nd of 256 channels, which are two blocks;
// `left` channels from the lane's first on.
__device__ __forceinline__ void quantize_strided(float (&y)[8], int left, uint8_t* codes, uint8_t* scales) {
  float amax[2];
  auto maxima = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      amax[h] = fmaxf(fmaxf(fabsf(y[4 * h]), fabsf(y[4 * h + 1])), fmaxf(fabsf(y[4 * h + 2]), fabsf(y[4 * h + 3])));
      amax[h] = fmaxf(amax[h], 0.f);  // (NaN alone counts nothing)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax[h] = fmaxf(amax[h], __shfl_xor_sync(0xffffffffu, amax[h], o));
    }
  };
  maxima();
  if (!fp8_is_finite(fmaxf(amax[0], amax[1]))) {  // infinities (rare): NaN, and out of the maxima
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (!fp8_is_finite(y[j])) y[j] = fp8_nan();
    maxima();
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int e = fp8_exponent(amax[h]);
    const float inv = fp8_pow2(-e);
#pragma unroll
    for (int j = 4 * h; j < 4 * h + 4; j += 2) {
      const uint32_t pair = fp8_pack2(y[j] * inv, y[j + 1] * inv);
      if (32 * j < left) codes[32 * j] = static_cast<uint8_t>(pair);
      if (32 * j + 32 < left) codes[32 * j + 32] = static_cast<uint8_t>(pair >> 8);
    }
    if (lane_id() == 0 && 128 * h < left) scales[h] = static_cast<uint8_t>(e + 127);
  }
}

// Blocks per SM: the kernel waits for memory, so as many as its registers
// allow (51201 x 1000 bf16: 73.4 us with four, 69.1 with five, 84 with six, which spill;
// 6400 x 256 f16: 4.1, 3.8 and 3.5 us).
constexpr int resident_blocks(int warps, int iters, int element_bytes) {
  return iters == 1 && element_bytes == 2 ? 6 : (warps == 1 && element_bytes == 2 ? 5 : 4);
}

// WARPS warps per row (1: eight rows per 256-thread block), ITERS x 8 channels a lane.
template <typename T, int WARPS, int ITERS, bool NORM, bool VEC>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : WARPS * 32,
                                  WARPS == 32 ? 1 : resident_blocks(WARPS, ITERS, sizeof(T)))
    fp8_rows_kernel(const RowsParams p) {
  __shared__ float s_part[WARPS == 1 ? 1 : WARPS];
  constexpr int kLanes = WARPS * 32;
  const int lane = lane_id(), in_row = WARPS == 1 ? 0 : warp_id();
  const int per_block = WARPS == 1 ? 8 : 1;
  // (unsigned: the last step may pass 2^31)
  const unsigned first_row = blockIdx.x * per_block + (WARPS == 1 ? threadIdx.x >> 5 : 0);
  const unsigned step = gridDim.x * per_block, rows = p.rows;

  pdl_begin();
  // gamma in shared memory: in registers it took a third of them, and half the
  // warps.  The first row's values come to L1 meanwhile.
  extern __shared__ float s_gamma[];
  if constexpr (NORM) {
    if (first_row < rows) {
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        const int c = channel_of<VEC>(i * WARPS + in_row, lane, 0);
        if (c >= p.channels) continue;
        prefetch_l1(static_cast<const T*>(p.x) + first_row * p.x_ld + c);
        if (p.residual) prefetch_l1(static_cast<const T*>(p.residual) + first_row * p.r_ld + c);
      }
    }
    const bool whole = p.gamma && p.channels % 4 == 0 && reinterpret_cast<uintptr_t>(p.gamma) % 16 == 0;
    for (int c = threadIdx.x * 4; c < ITERS * kLanes * 8; c += blockDim.x * 4) {
      float4 g = make_float4(1.f, 1.f, 1.f, 1.f);
      if (whole) {
        if (c < p.channels) g = *reinterpret_cast<const float4*>(p.gamma + c);
      } else if (p.gamma) {
        float* e = &g.x;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < p.channels) e[k] = p.gamma[c + k];
      }
      *reinterpret_cast<float4*>(s_gamma + c) = g;
    }
    __syncthreads();
  }
  for (unsigned row = first_row; row < rows; row += step) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
    const T* r = static_cast<const T*>(p.residual) + (p.residual ? row * p.r_ld : 0);
    float v[ITERS][8];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      const int warp = i * WARPS + in_row;
      if (channel_of<VEC>(warp, lane, 0) < p.channels) {
        load_row8<T, VEC>(x, warp, lane, p.channels, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      }
    }
    if (p.residual) {
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        const int warp = i * WARPS + in_row;
        if (channel_of<VEC>(warp, lane, 0) < p.channels) {
          float a[8];
          load_row8<T, VEC>(r, warp, lane, p.channels, a);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] += a[j];
        }
      }
    }
    if (p.h) {
      T* h = static_cast<T*>(p.h) + row * p.h_ld;
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        const int warp = i * WARPS + in_row;
        if constexpr (VEC) {
          const int c = channel_of<VEC>(warp, lane, 0);
          if (c < p.channels) store8<T>(h + c, v[i]);
        } else {
          T* at = h + channel_of<VEC>(warp, lane, 0);
          const int left = p.channels - channel_of<VEC>(warp, lane, 0);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (32 * j < left) at[32 * j] = from_f32<T>(v[i][j]);
        }
      }
    }
    if constexpr (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < ITERS; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[i][j], v[i][j], sum);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if constexpr (WARPS > 1) {
        if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) sum += s_part[w];
        __syncthreads();  // before the next row's partial sums
      }
      const float rstd = rsqrtf(sum / static_cast<float>(p.channels) + p.eps);
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        const int warp = i * WARPS + in_row;
        float g[8];
        if constexpr (VEC) {
          load8<float>(s_gamma + channel_of<VEC>(warp, lane, 0), g);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) g[j] = s_gamma[channel_of<VEC>(warp, lane, j)];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * rstd * g[j];
      }
    }
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      const int c = channel_of<VEC>(i * WARPS + in_row, lane, 0);
      uint8_t* codes = p.codes + row * p.codes_ld + c;
      uint8_t* scales = p.scales + row * p.scales_ld + c / kFp8Block;
      if constexpr (VEC) {
        quantize_block(v[i], c < p.channels, c % kFp8Block == 0, codes, scales);
      } else {
        quantize_strided(v[i], p.channels - c, codes, scales);
      }
    }
  }
}

template <typename T, bool NORM, bool VEC>
int launch_rows(cudaStream_t stream, const RowsParams& p, const char* what) {
  const int sms = sm_count();
  const int c = p.channels;
  // A resident grid; rows beyond it are walked by the same blocks.
  auto smem = [](int lanes, int iters) { return NORM ? static_cast<size_t>(lanes) * iters * 8 * sizeof(float) : 0; };
  if (c <= 1024) {
    const int iters = c <= 256 ? 1 : (c <= 512 ? 2 : 4);
    const int blocks = std::min((p.rows - 1) / 8 + 1, sms * resident_blocks(1, iters, sizeof(T)));
    auto k = iters == 1 ? fp8_rows_kernel<T, 1, 1, NORM, VEC>
                        : (iters == 2 ? fp8_rows_kernel<T, 1, 2, NORM, VEC> : fp8_rows_kernel<T, 1, 4, NORM, VEC>);
    return launch_kernel(k, dim3(blocks), dim3(256), smem(32, iters), stream, what, p);
  }
  if (c <= 8192) {
    const int iters = c <= 2048 ? 1 : (c <= 4096 ? 2 : 4);
    const int blocks = std::min(p.rows, sms * resident_blocks(8, iters, sizeof(T)));
    auto k = iters == 1 ? fp8_rows_kernel<T, 8, 1, NORM, VEC>
                        : (iters == 2 ? fp8_rows_kernel<T, 8, 2, NORM, VEC> : fp8_rows_kernel<T, 8, 4, NORM, VEC>);
    return launch_kernel(k, dim3(blocks), dim3(256), smem(256, iters), stream, what, p);
  }
  static unsigned long long configured = 0;
  auto k = fp8_rows_kernel<T, 32, 4, NORM, VEC>;
  const int rc =
      ensure_smem_attribute(reinterpret_cast<const void*>(k), static_cast<int>(smem(1024, 4)), &configured, what);
  if (rc != LDB_OK) return rc;
  return launch_kernel(k, dim3(std::min(p.rows, sms)), dim3(1024), smem(1024, 4), stream, what, p);
}

template <typename T>
int launch_vec(cudaStream_t stream, const RowsParams& p, bool norm, bool vec, const char* what) {
  if (norm) return vec ? launch_rows<T, true, true>(stream, p, what) : launch_rows<T, true, false>(stream, p, what);
  return vec ? launch_rows<T, false, true>(stream, p, what) : launch_rows<T, false, false>(stream, p, what);
}

int esize(int dtype) { return dtype == LDB_F32 ? 4 : 2; }

bool aligned16(const void* p, long long ld, int es) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0);
}

int run_rows(cudaStream_t stream, RowsParams p, int dtype, bool norm, const char* what) {
  if (p.rows != 0 && (!p.x || !p.codes || !p.scales)) return fail(LDB_ERR_INVALID, "%s: null pointer", what);
  if (dtype != LDB_F16 && dtype != LDB_F32 && dtype != LDB_BF16)
    return fail(LDB_ERR_INVALID, "%s: unknown element type %d", what, dtype);
  if (p.rows < 0 || p.channels <= 0 || p.channels > 32768)
    return fail(LDB_ERR_SHAPE, "%s: %d rows of %d channels (1..32768)", what, p.rows, p.channels);
  const int blocks = (p.channels + kFp8Block - 1) / kFp8Block;
  if (p.x_ld < p.channels || (p.residual && p.r_ld < p.channels) || (p.h && p.h_ld < p.channels) ||
      p.codes_ld < p.channels || p.scales_ld < blocks)
    return fail(LDB_ERR_SHAPE, "%s: a row stride is shorter than its row", what);
  if (p.codes_ld % 16 || reinterpret_cast<uintptr_t>(p.codes) % 16)
    return fail(LDB_ERR_ALIGNMENT, "%s: codes need 16-byte aligned rows", what);
  if (p.rows == 0) return LDB_OK;
  const int es = esize(dtype);
  const bool vec = p.channels % 8 == 0 && aligned16(p.x, p.x_ld, es) && aligned16(p.residual, p.r_ld, es) &&
                   aligned16(p.h, p.h_ld, es);
  if (dtype == LDB_F16) return launch_vec<__half>(stream, p, norm, vec, what);
  if (dtype == LDB_BF16) return launch_vec<__nv_bfloat16>(stream, p, norm, vec, what);
  return launch_vec<float>(stream, p, norm, vec, what);
}

// One 128 x 128 block of a weight: eight warps, 16 rows each, four columns a
// lane held in registers between the maximum and the rounding.  Runs once per
// weight; not tuned.
template <typename T>
__global__ void __launch_bounds__(256) fp8_pack_weight_kernel(const T* w, long long w_ld, int n, int k, uint8_t* codes,
                                                              long long codes_ld, uint8_t* scales, int scales_ld) {
  __shared__ float s_max[8];
  pdl_begin();
  const int warp = warp_id(), lane = lane_id();
  const int col = blockIdx.x * kFp8Block + lane * 4;
  float v[16][4];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = blockIdx.y * kFp8Block + i * 8 + warp;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = row < n && col + j < k ? to_f32<T>(w[row * w_ld + col + j]) : 0.f;
      if (!fp8_is_finite(a)) a = fp8_nan();
      v[i][j] = a;
      amax = fmaxf(amax, fabsf(a));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (lane == 0) s_max[warp] = amax;
  __syncthreads();
  amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, s_max[i]);
  const int e = fp8_exponent(amax);
  const float inv = fp8_pow2(-e);
  if (threadIdx.x == 0)
    scales[static_cast<long long>(blockIdx.y) * scales_ld + blockIdx.x] = static_cast<uint8_t>(e + 127);
  if (col >= k) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = blockIdx.y * kFp8Block + i * 8 + warp;
    if (row < n)
      *reinterpret_cast<uint32_t*>(codes + row * codes_ld + col) =
          fp8_pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
  }
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_rms_norm_fp8(cudaStream_t stream, const void* x, long long x_ld, const void* residual, long long residual_ld,
                     int dtype, const float* gamma, float eps, void* h, long long h_ld, uint8_t* codes,
                     long long codes_ld, uint8_t* scales, long long scales_ld, int rows, int channels) {
  ldb::RowsParams p{x, residual, gamma, h, codes, scales, x_ld, residual_ld, h_ld, codes_ld, scales_ld,
                    rows, channels, eps};
  return ldb::run_rows(stream, p, dtype, true, "rms_norm_fp8");
}

int ldb_quantize_fp8_rows(cudaStream_t stream, const void* x, long long x_ld, int dtype, uint8_t* codes,
                          long long codes_ld, uint8_t* scales, long long scales_ld, int rows, int channels) {
  ldb::RowsParams p{x, nullptr, nullptr, nullptr, codes, scales, x_ld, 0, 0, codes_ld, scales_ld,
                    rows, channels, 0.f};
  return ldb::run_rows(stream, p, dtype, false, "quantize_fp8_rows");
}

int ldb_pack_weight_fp8(cudaStream_t stream, const void* w, long long w_ld, int dtype, uint8_t* codes,
                        long long codes_ld, uint8_t* scales, int scales_ld, int n, int k) {
  using namespace ldb;
  if (!w || !codes || !scales) return fail(LDB_ERR_INVALID, "pack_weight_fp8: null pointer");
  if (dtype != LDB_F16 && dtype != LDB_F32 && dtype != LDB_BF16)
    return fail(LDB_ERR_INVALID, "pack_weight_fp8: unknown element type %d", dtype);
  if (n <= 0 || k <= 0) return fail(LDB_ERR_SHAPE, "pack_weight_fp8: %d x %d", n, k);
  const int kb = (k + kFp8Block - 1) / kFp8Block, nb = (n + kFp8Block - 1) / kFp8Block;
  if (w_ld < k || codes_ld < k || scales_ld < kb)
    return fail(LDB_ERR_SHAPE, "pack_weight_fp8: a row stride is shorter than its row");
  if (nb > 65535) return fail(LDB_ERR_SHAPE, "pack_weight_fp8: at most 8388480 rows");
  if (codes_ld % 16 || reinterpret_cast<uintptr_t>(codes) % 16)
    return fail(LDB_ERR_ALIGNMENT, "pack_weight_fp8: codes need 16-byte aligned rows");
  const dim3 grid(kb, nb);
  const char* what = "pack_weight_fp8 launch";
  if (dtype == LDB_F16)
    return launch_kernel(fp8_pack_weight_kernel<__half>, grid, dim3(256), 0, stream, what,
                         static_cast<const __half*>(w), w_ld, n, k, codes, codes_ld, scales, scales_ld);
  if (dtype == LDB_BF16)
    return launch_kernel(fp8_pack_weight_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, what,
                         static_cast<const __nv_bfloat16*>(w), w_ld, n, k, codes, codes_ld, scales, scales_ld);
  return launch_kernel(fp8_pack_weight_kernel<float>, grid, dim3(256), 0, stream, what, static_cast<const float*>(w),
                       w_ld, n, k, codes, codes_ld, scales, scales_ld);
}

}  // extern "C"
