// Writing new tokens into the paged 8-bit key/value cache.
//
// One warp or block per touched (page, kv head) of K or V.  With `held` older tokens in
// the page and e(new) the scale that the new values need (fp8.cuh):
//
//   e = held > 0 ? max(e_old, e(new)) : e(new)     within -96 .. 96
//   new codes = e4m3(x 2^-e);  if e > e_old, old codes = e4m3(code 2^(e_old - e))
//
// so a page that is filled token by token keeps one scale, and what it holds is
// rounded again only when that scale grows.  New values without a finite one other than
// zero have no e(new) there: with the scale 1 that they have in a page of their own, a
// padded token would make a page of scale 2^-9 512 times as coarse.  Writing the same
// tokens at the same place again changes nothing.
//
// Bound: HBM (2 bytes read and 1 written a value); a page's new values stay in
// registers between the maximum and the rounding.  For one token it is the
// launch.  One B200: 4 x 2049 tokens of 8 x 128 bf16 13.1 us (3.8 TB/s: a unit's
// reads depend on one another, and the grid is not many times what is
// resident), one token of 32 items 2.6 us.

#include <type_traits>

#include "host_common.h"
#include "kv_cache.cuh"

namespace ldb {
namespace {

struct AppendParams {
  const void* src[2];      // new keys, new values
  uint8_t* codes[2];
  uint8_t* scales[2];
  const int* table;
  const int* start;        // [batch] first position written
  const int* counts;       // [batch] tokens written, null: all `tokens`
  long long src_ld[2], src_batch[2], table_ld;
  int pages, kv_heads, page, width, dim, dim_shift, tokens;
  int vec;  // 16-byte reads of eight values
};

constexpr int kAppendThreads = 256;
constexpr int kMaxVecs = 8;  // vectors of eight per thread

// The largest value of a unit's threads.
template <int WARPS>
__device__ __forceinline__ float unit_max(float v, float* s_part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (WARPS > 1) {
    __syncthreads();
    if (lane_id() == 0) s_part[warp_id()] = v;
    __syncthreads();
    v = s_part[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) v = fmaxf(v, s_part[w]);
  }
  return v;
}

// Largest magnitude of eight values (NaN left out), two at a time in 16 bits.
template <typename T>
__device__ __forceinline__ float max_of8(const uint4 (&raw)[sizeof(T) / 2]) {
  if constexpr (sizeof(T) == 4) {
    const float* v = reinterpret_cast<const float*>(raw);
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* v = reinterpret_cast<const T2*>(raw);
    const T2 m = __hmax2(__hmax2(__habs2(v[0]), __habs2(v[1])), __hmax2(__habs2(v[2]), __habs2(v[3])));
    const float a = to_f32<T>(m.x), b = to_f32<T>(m.y);
    return fmaxf(fmaxf(a, b), 0.f);  // (a NaN, left where all are one, counts nothing)
  }
}

// WARPS of a unit (a page of one head), VECS vectors of eight values per thread
// that a whole page takes: a warp up to 256 vectors, eight units to a block, and a
// unit a block above.  (4 x 2049 tokens, 8 heads of 64 in pages of 16: 19.2 us with 256
// threads a unit, 6.9 so.)  Above 256 vectors a thread takes eight of them where a call has
// fewer tokens than a page, which leaves most threads of a unit without work: one token of 32
// items, 8 heads of 128 in pages of 64, 2.5 us with eight and 4.5 with four, 8 tokens of 64
// items 6.4 and 8.4.  Else four, up to 1024 vectors, us with eight and with four: pages of 512
// vectors 3.0 and 2.2 (128 tokens, 8 heads of 128), 6.3 and 5.0 (16 x 600, 2 heads of 128), 13.2
// and 12.4 (4 x 2049, 8 of 128), 4.6 and 5.4 (the same, of 32); of 1024 3.0 and 2.3,
// 6.2 and 5.1, 13.2 and 13.2, 7.0 and 7.3 (of 64); of 2048 3.1 and 2.8, 6.4 and 6.7, 13.7
// and 13.8.  The values stay as they came (four registers a vector in 16 bits) until
// they are rounded, so that enough warps are resident to cover the chain of
// dependent reads (position, page number, values).
template <typename T, int VECS, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? kAppendThreads : WARPS * 32,
                                  (sizeof(T) == 4 ? 3 : (VECS == kMaxVecs ? 4 : 6)) * (WARPS == 1 ? 1 : 8 / WARPS))
    kv_append_kernel(const AppendParams p, unsigned int* status) {
  constexpr int kUnitThreads = WARPS * 32;
  __shared__ float s_part[kAppendThreads / 32];
  pdl_begin();
  const int thread = WARPS == 1 ? lane_id() : threadIdx.x;
  const int u = WARPS == 1 ? blockIdx.x * (kAppendThreads / 32) + warp_id() : blockIdx.x;
  const int b = blockIdx.y, head = u % p.kv_heads, which = blockIdx.z;
  const int start = p.start[b];
  int count = p.counts ? p.counts[b] : p.tokens;
  if (start < 0 || count < 0 || count > p.tokens) {
    if (thread == 0) set_bad_shape(status);
    return;
  }
  const long long slot = static_cast<long long>(start / p.page) + u / p.kv_heads;
  const long long page0 = slot * p.page;
  const int first = static_cast<int>(max(0ll, page0 - start));                              // of the new tokens
  const int last = static_cast<int>(min(static_cast<long long>(count), page0 + p.page - start));
  if (first >= last) return;
  const int held = static_cast<int>(max(0ll, start - page0));
  const int id = slot < p.width ? p.table[b * p.table_ld + slot] : -1;  // (looked at once the values are on their way)
  const T* src = static_cast<const T*>(p.src[which]) + b * p.src_batch[which] + head * p.dim;
  const int vshift = p.dim_shift - 3;  // vectors of eight per token
  const int vecs = (last - first) << vshift;

  uint4 raw[VECS][sizeof(T) / 2];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int q = i * kUnitThreads + thread;
    if (q < vecs) {
      const T* x = src + (first + (q >> vshift)) * p.src_ld[which] + ((q & ((1 << vshift) - 1)) << 3);
      if (p.vec) {
#pragma unroll
        for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h) raw[i][h] = reinterpret_cast<const uint4*>(x)[h];
      } else {
        T t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = x[j];
#pragma unroll
        for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h) raw[i][h] = reinterpret_cast<const uint4*>(t)[h];
      }
    }
  }
  if (id < 0 || id >= p.pages) {
    if (thread == 0) set_bad_shape(status);
    return;
  }
  const long long unit = static_cast<long long>(id) * p.kv_heads + head;
  uint8_t* codes = p.codes[which] + unit * p.page * p.dim;
  uint8_t* scale = p.scales[which] + unit;
  const int old_scale = held > 0 ? *scale : 127;
#pragma unroll
  for (int i = 0; i < VECS; ++i)
    if (i * kUnitThreads + thread < vecs) amax = fmaxf(amax, max_of8<T>(raw[i]));
  amax = unit_max<WARPS>(amax, s_part);
  const bool infinite = !fp8_is_finite(amax);  // (rare: infinities become NaN and leave the maximum)
  if (infinite) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      if (i * kUnitThreads + thread < vecs) {
        const T* v = reinterpret_cast<const T*>(raw[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = fabsf(to_f32<T>(v[j]));
          if (fp8_is_finite(a)) amax = fmaxf(amax, a);
        }
      }
    }
    amax = unit_max<WARPS>(amax, s_part);
  }
  const int e_old = old_scale - 127;
  int e = max(-kKvMaxExponent, min(kKvMaxExponent, fp8_exponent(amax)));
  if (held > 0) e = amax == 0.f ? e_old : max(e, e_old);  // zeros ask for no scale
  const float inv = fp8_pow2(-min(e, 127));
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int q = i * kUnitThreads + thread;
    if (q < vecs) {
      const T* v = reinterpret_cast<const T*>(raw[i]);
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = to_f32<T>(v[j]) * inv;
        if (infinite && !fp8_is_finite(y[j])) y[j] = fp8_nan();
      }
      uint2 packed;
      packed.x = fp8_pack4(y[0], y[1], y[2], y[3]);
      packed.y = fp8_pack4(y[4], y[5], y[6], y[7]);
      *reinterpret_cast<uint2*>(codes + ((static_cast<long long>(held) << p.dim_shift) + (q << 3))) = packed;
    }
  }
  if (held > 0 && e > e_old) {
    const float shrink = exp2f(static_cast<float>(max(e_old - e, -64)));  // below 2^-18 every code becomes 0
    for (int q = thread; q < held << vshift; q += kUnitThreads) {
      uint2* at = reinterpret_cast<uint2*>(codes + (q << 3));
      uint2 old = *at;
      uint32_t* w = &old.x;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t word = h == 0 ? old.x : old.y;
        const uint32_t lo = fp8_unpack2(word & 0xFFFFu), hi = fp8_unpack2(word >> 16);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        w[h] = fp8_pack4(a.x * shrink, a.y * shrink, c.x * shrink, c.y * shrink);
      }
      *at = old;
    }
  }
  if (WARPS == 1) __syncwarp();  // all have read the old one
  if (thread == 0) *scale = static_cast<uint8_t>(e + 127);
}

template <typename T>
int launch_append(cudaStream_t stream, long long units, int batch, const AppendParams& p, unsigned int* status) {
  const int vecs = p.page * p.dim / 8;  // 64 .. 2048, a power of two
  const bool four = p.tokens >= p.page;  // vectors a thread, from 512 to 1024 a page
  auto k = vecs <= 64    ? kv_append_kernel<T, 2, 1>
           : vecs <= 128 ? kv_append_kernel<T, 4, 1>
           : vecs <= 256 ? kv_append_kernel<T, kMaxVecs, 1>
           : vecs <= 512 ? (four ? kv_append_kernel<T, 4, 4> : kv_append_kernel<T, kMaxVecs, 2>)
           : vecs <= 1024 ? (four ? kv_append_kernel<T, 4, 8> : kv_append_kernel<T, kMaxVecs, 4>)
                          : kv_append_kernel<T, kMaxVecs, 8>;
  const long long blocks = vecs <= 256 ? (units + kAppendThreads / 32 - 1) / (kAppendThreads / 32) : units;
  if (blocks > 0x7FFFFFFFll || units > 0x7FFFFF00ll)
    return fail(LDB_ERR_SHAPE, "kv_append: %lld pages and heads of an item", units);
  const dim3 grid(static_cast<unsigned>(blocks), batch, 2);
  const int threads = vecs <= 256 ? kAppendThreads : vecs / (four && vecs <= 1024 ? 4 : kMaxVecs);
  return launch_kernel(k, grid, dim3(threads), 0, stream, "kv_append launch", p, status);
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_kv_append_fp8(cudaStream_t stream, const void* k, long long k_ld, long long k_batch, const void* v,
                      long long v_ld, long long v_batch, int dtype, uint8_t* k_codes, uint8_t* v_codes,
                      uint8_t* k_scales, uint8_t* v_scales, int pages, int kv_heads, int page, int head_dim,
                      const int* table, long long table_ld, int width, const int* start, const int* counts, int batch,
                      int tokens) {
  using namespace ldb;
  if (batch < 0 || tokens < 0) return fail(LDB_ERR_SHAPE, "kv_append: %d items of %d tokens", batch, tokens);
  if (dtype != LDB_F16 && dtype != LDB_F32 && dtype != LDB_BF16)
    return fail(LDB_ERR_INVALID, "kv_append: unknown element type %d", dtype);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(LDB_ERR_SHAPE, "kv_append: head_dim %d (32, 64 or 128)", head_dim);
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return fail(LDB_ERR_SHAPE, "kv_append: pages of %d tokens (16, 32, 64 or 128)", page);
  if (pages <= 0 || kv_heads <= 0 || width <= 0 || table_ld < width)
    return fail(LDB_ERR_SHAPE, "kv_append: %d pages, %d heads, table of %d", pages, kv_heads, width);
  if (batch == 0 || tokens == 0) return LDB_OK;
  if (!k || !v || !k_codes || !v_codes || !k_scales || !v_scales || !table || !start)
    return fail(LDB_ERR_INVALID, "kv_append: null pointer");
  const long long row = static_cast<long long>(kv_heads) * head_dim;
  if ((tokens > 1 && (k_ld < row || v_ld < row)) || static_cast<long long>(batch) * kv_heads > 65535)
    return fail(LDB_ERR_SHAPE, "kv_append: row strides below %lld, or more than 65535 (item, head) pairs", row);
  if (reinterpret_cast<uintptr_t>(k_codes) % 16 || reinterpret_cast<uintptr_t>(v_codes) % 16)
    return fail(LDB_ERR_ALIGNMENT, "kv_append: codes must be 16-byte aligned");
  unsigned int* status = device_status_ptr();
  if (!status) return fail(LDB_ERR_CUDA, "kv_append: no device status word");
  AppendParams p{};
  p.src[0] = k, p.src[1] = v, p.codes[0] = k_codes, p.codes[1] = v_codes;
  p.scales[0] = k_scales, p.scales[1] = v_scales;
  p.src_ld[0] = k_ld, p.src_ld[1] = v_ld, p.src_batch[0] = k_batch, p.src_batch[1] = v_batch;
  p.table = table, p.table_ld = table_ld, p.start = start, p.counts = counts;
  p.pages = pages, p.kv_heads = kv_heads, p.page = page, p.width = width, p.dim = head_dim;
  p.dim_shift = head_dim == 32 ? 5 : (head_dim == 64 ? 6 : 7);
  p.tokens = tokens;
  const int es = dtype == LDB_F32 ? 4 : 2;
  p.vec = 1;
  for (int i = 0; i < 2; ++i)
    if (reinterpret_cast<uintptr_t>(p.src[i]) % 16 || p.src_ld[i] * es % 16 || p.src_batch[i] * es % 16) p.vec = 0;
  // pages that a run of `tokens` can touch, wherever it starts
  const long long touched = (static_cast<long long>(tokens) + page - 2) / page + 1;
  const long long units = touched * kv_heads;
  if (dtype == LDB_F16) return launch_append<__half>(stream, units, batch, p, status);
  if (dtype == LDB_BF16) return launch_append<__nv_bfloat16>(stream, units, batch, p, status);
  return launch_append<float>(stream, units, batch, p, status);
}

}  // extern "C"
