// Writing new tokens into the paged 4-bit key/value cache.
//
//   s = least scale with max|x| <= 7.5 s over 16 channels;  code = rn(x / s) + 8
//
// A token's scales are its own, so nothing that the pages hold is read or
// rounded again and tokens can be written in any order.  A thread takes one group of
// channels of four neighbouring tokens of a page: their scales are one word,
// neighbouring threads read neighbouring groups (whole rows of all heads) and four
// reads are on their way at a time.
//
// Bound: HBM, 2 bytes read and 9/16 written a value; for one token the launch.  One B200, 4 x 4097
// tokens of 8 heads of 128 bf16 with the read back that follows 35 us (172 MB at 4.9 TB/s), one token of 32 items with its
// read back 3.9 us.  Eight channels a thread instead of a group find each group's maximum twice, and took longer.

#include <type_traits>

#include "host_common.h"
#include "kv_int4.cuh"

namespace ldb {
namespace {

struct AppendParams {
  const void* src[2];  // new keys, new values
  uint8_t* codes[2];
  uint8_t* scales[2];
  const int* table;
  const int* start;    // [batch] first position written
  const int* counts;   // [batch] tokens written, null: all `tokens`
  long long src_ld[2], src_batch[2], table_ld;
  int pages, kv_heads, page_shift, width, dim, group_shift, tokens;
  int vec;  // 16-byte reads of eight values
};

constexpr int kThreads = 128;

// The largest magnitude of a group, infinite where one is not finite.
template <typename T>
__device__ __forceinline__ float largest16(const uint4 (&raw)[sizeof(T)]) {
  constexpr uint32_t kSign = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
  uint32_t m = 0;  // (magnitudes order as their bits do)
#pragma unroll
  for (int h = 0; h < static_cast<int>(sizeof(T)); ++h) {
    const uint32_t w[4] = {raw[h].x, raw[h].y, raw[h].z, raw[h].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) m = sizeof(T) == 4 ? max(m, w[k] & kSign) : __vmaxu2(m, w[k] & kSign);
  }
  if constexpr (sizeof(T) == 4) return __uint_as_float(min(m, 0x7F800000u));
  constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  const uint32_t top = min(max(m & 0xFFFFu, m >> 16), kInf);
  return std::is_same<T, __half>::value ? __half2float(__ushort_as_half(static_cast<unsigned short>(top)))
                                        : __uint_as_float(top << 16);
}

// A group's values in FP32, in pairs of neighbours.
template <typename T>
__device__ __forceinline__ void pairs16(const uint4 (&raw)[sizeof(T)], uint64_t (&x)[2][4]) {
  constexpr int kWords = 4 * sizeof(T);
  uint32_t w[kWords];
#pragma unroll
  for (int h = 0; h < static_cast<int>(sizeof(T)); ++h)
    w[4 * h] = raw[h].x, w[4 * h + 1] = raw[h].y, w[4 * h + 2] = raw[h].z, w[4 * h + 3] = raw[h].w;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (sizeof(T) == 4) {
      x[k / 4][k % 4] = pack2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[k / 4][k % 4] = pack2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u));
    } else {
      const float2 f = __half22float2(as_half2(w[k]));
      x[k / 4][k % 4] = pack2(f.x, f.y);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) kv_append_int4_kernel(const AppendParams p, unsigned int* status) {
  pdl_begin();
  const int b = blockIdx.y, which = blockIdx.z;
  const unsigned per = static_cast<unsigned>(p.kv_heads) << p.group_shift;  // groups of a token
  const unsigned u = blockIdx.x * kThreads + threadIdx.x;
  const unsigned quad = u / per, rest = u - quad * per;
  const int head = rest >> p.group_shift, group = rest & ((1 << p.group_shift) - 1);
  const int start = p.start[b];
  const int count = p.counts ? p.counts[b] : p.tokens;
  if (start < 0 || count < 0 || count > p.tokens) {
    if (u == 0) set_bad_shape(status);
    return;
  }
  const long long at0 = static_cast<long long>(start & ~(kInt4Quad - 1)) + static_cast<long long>(quad) * kInt4Quad;
  const int first = static_cast<int>(max(0ll, start - at0));  // of the quad's tokens
  const int last = static_cast<int>(min(static_cast<long long>(kInt4Quad), static_cast<long long>(start) + count - at0));
  if (first >= last) return;
  const long long slot = at0 >> p.page_shift;
  const int id = slot < p.width ? p.table[b * p.table_ld + slot] : -1;  // (looked at once the values are on their way)
  const T* src = static_cast<const T*>(p.src[which]) + b * p.src_batch[which] + rest * kInt4Group +
                 (at0 - start) * p.src_ld[which];
  uint4 raw[kInt4Quad][sizeof(T)];
#pragma unroll
  for (int j = 0; j < kInt4Quad; ++j) {
    if (j < first || j >= last) continue;
    const T* x = src + j * p.src_ld[which];
    if (p.vec) {
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(T)); ++h) raw[j][h] = reinterpret_cast<const uint4*>(x)[h];
    } else {
      __align__(16) T t[kInt4Group];
#pragma unroll
      for (int c = 0; c < kInt4Group; ++c) t[c] = x[c];
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(T)); ++h) raw[j][h] = reinterpret_cast<const uint4*>(t)[h];
    }
  }
  if (id < 0 || id >= p.pages) {
    set_bad_shape(status);
    return;
  }
  const int in_page = static_cast<int>(at0 & ((1 << p.page_shift) - 1));
  const long long unit = static_cast<long long>(id) * p.kv_heads + head;
  uint8_t* codes = p.codes[which] + ((unit << p.page_shift) + in_page) * (p.dim / 2) + group * (kInt4Group / 2);
  uint8_t* scale = p.scales[which] + ((((unit << p.group_shift) + group) << p.page_shift) + in_page);
  uint32_t bytes = 0;
#pragma unroll
  for (int j = 0; j < kInt4Quad; ++j) {
    if (j < first || j >= last) continue;
    const float amax = largest16<T>(raw[j]);
    const bool finite = fp8_is_finite(amax);
    const int byte = finite ? int4_scale_byte(amax) : kInt4NanScale;
    const Int4Inverse inv(byte);
    uint64_t x[2][4];
    pairs16<T>(raw[j], x);
    if (byte >= kInt4TopScale) {  // (rare) past the scales' end, or not finite
      const float most = finite ? 8.f * int4_scale_value(byte) : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float a, c;
        unpack2(x[k / 4][k % 4], a, c);
        x[k / 4][k % 4] = finite ? pack2(fmaxf(a, -most), fmaxf(c, -most)) : 0;
      }
    }
    *reinterpret_cast<uint2*>(codes + j * (p.dim / 2)) = make_uint2(int4_pack8(x[0], inv), int4_pack8(x[1], inv));
    bytes |= static_cast<uint32_t>(byte) << (8 * j);
  }
  if (last - first == kInt4Quad) {
    *reinterpret_cast<uint32_t*>(scale) = bytes;
  } else {
#pragma unroll
    for (int j = 0; j < kInt4Quad; ++j)
      if (j >= first && j < last) scale[j] = static_cast<uint8_t>(bytes >> (8 * j));
  }
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_kv_append_int4(cudaStream_t stream, const ldb_kv_append_desc* desc) {
  using namespace ldb;
  if (const int rc = check_desc(desc, "kv_append")) return rc;
  const auto& [struct_size, dtype, cache, k, v, k_ld, k_batch, v_ld, v_batch, start, counts, tokens] = *desc;
  const auto& [k_codes, v_codes, k_scales, v_scales, table, table_ld, pages, kv_heads, page, head_dim, width, batch] =
      cache;
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
  const long long groups = row / kInt4Group;
  // quads that a run of `tokens` can touch, wherever it starts
  const long long units = ((static_cast<long long>(tokens) + kInt4Quad - 2) / kInt4Quad + 1) * groups;
  if ((tokens > 1 && (k_ld < row || v_ld < row)) || batch > 65535 || units > 0x7FFFFF00ll)
    return fail(LDB_ERR_SHAPE, "kv_append: row strides below %lld, more than 65535 items, or %lld channels and tokens",
                row, units);
  for (const uint8_t* t : {k_codes, v_codes, k_scales, v_scales})
    if (reinterpret_cast<uintptr_t>(t) % 16)
      return fail(LDB_ERR_ALIGNMENT, "kv_append: codes and scales must be 16-byte aligned");
  unsigned int* status = device_status_ptr();
  if (!status) return fail(LDB_ERR_CUDA, "kv_append: no device status word");
  AppendParams p{};
  p.src[0] = k, p.src[1] = v, p.codes[0] = k_codes, p.codes[1] = v_codes;
  p.scales[0] = k_scales, p.scales[1] = v_scales;
  p.src_ld[0] = k_ld, p.src_ld[1] = v_ld, p.src_batch[0] = k_batch, p.src_batch[1] = v_batch;
  p.table = table, p.table_ld = table_ld, p.start = start, p.counts = counts;
  p.pages = pages, p.kv_heads = kv_heads, p.width = width, p.dim = head_dim, p.tokens = tokens;
  p.page_shift = page == 16 ? 4 : (page == 32 ? 5 : (page == 64 ? 6 : 7));
  p.group_shift = head_dim == 32 ? 1 : (head_dim == 64 ? 2 : 3);
  const int es = dtype == LDB_F32 ? 4 : 2;
  p.vec = 1;
  for (int i = 0; i < 2; ++i)
    if (reinterpret_cast<uintptr_t>(p.src[i]) % 16 || p.src_ld[i] * es % 16 || p.src_batch[i] * es % 16) p.vec = 0;
  auto kernel = dtype == LDB_F16    ? kv_append_int4_kernel<__half>
                : dtype == LDB_BF16 ? kv_append_int4_kernel<__nv_bfloat16>
                                    : kv_append_int4_kernel<float>;
  const dim3 grid(static_cast<unsigned>((units + kThreads - 1) / kThreads), batch, 2);
  return launch_kernel(kernel, grid, dim3(kThreads), 0, stream, "kv_append launch", p, status);
}

}  // extern "C"
