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
// Bound: HBM, 2 bytes read and 9/16 written a value; for one token the launch.

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
      T t[kInt4Group];
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
    float x[2][8];
    const T* v = reinterpret_cast<const T*>(raw[j]);
    float amax = 0.f;
    bool finite = true;
#pragma unroll
    for (int c = 0; c < kInt4Group; ++c) {
      x[c / 8][c % 8] = to_f32<T>(v[c]);
      amax = fmaxf(amax, fabsf(x[c / 8][c % 8]));
      finite = finite && fp8_is_finite(x[c / 8][c % 8]);
    }
    const int byte = finite ? int4_scale_byte(amax) : kInt4NanScale;
    const Int4Inverse inv(byte);
    if (!finite) {
#pragma unroll
      for (int c = 0; c < kInt4Group; ++c) x[c / 8][c % 8] = 0.f;
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

int ldb_kv_append_int4(cudaStream_t stream, const void* k, long long k_ld, long long k_batch, const void* v,
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
