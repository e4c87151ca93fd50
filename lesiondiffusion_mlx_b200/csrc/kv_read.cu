// Reading tokens of a paged key/value cache back as rows.
//
//   out[b, i] = value of item b's token start[b] + i where that lies below
//   lengths[b], else zeros
//
// from 4 bits ((code - 8) s, exact in every output type) or from e4m3 with the
// page's scale (rounded once).  A thread takes eight channels of four
// neighbouring tokens of a page: the 4-bit cache's scales of four are a word, and the stores of a warp
// are whole sectors (with 16 channels a thread, 32 bytes in two halves, items of up to 16384
// tokens took 137 us instead of 93, and with 8 or 16 tokens a thread 96).
//
// Bound: HBM, 9/16 or 1 byte read and 2 written a value.  One B200, 8 items of up to 16384 tokens, 8 heads
// of 128 in 4 bits: 93 us (610 MB at 6.5 TB/s); 77 tokens of 4 items of 4 heads of 64 in 8 bits 2.3 us.

#include <type_traits>

#include "host_common.h"
#include "kv_cache.cuh"
#include "kv_int4.cuh"

namespace ldb {
namespace {

struct ReadParams {
  const uint8_t* codes[2];
  const uint8_t* scales[2];
  void* out[2];
  const int* table;
  const int* lengths;
  const int* start;  // [batch] first token read, null: 0
  long long out_ld[2], out_batch[2], table_ld;
  int pages, kv_heads, page_shift, width, dim, group_shift, tokens;
  int vec;  // 16-byte stores
};

constexpr int kThreads = 128;

// Eight f16 values in order to the output's type.
template <typename T>
__device__ __forceinline__ void store_half8(T* to, const uint32_t (&v)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
    *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
  } else {
    float f[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = __half22float2(as_half2(v[k]));
      f[2 * k] = x.x, f[2 * k + 1] = x.y;
    }
    store8<T>(to, f);
  }
}

template <typename T, bool INT4>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const ReadParams p, unsigned int* status) {
  pdl_begin();
  const int b = blockIdx.y, which = blockIdx.z;
  const int shift = p.group_shift + 1;  // eights of a head's channels
  const unsigned per = static_cast<unsigned>(p.kv_heads) << shift;
  const unsigned u = blockIdx.x * kThreads + threadIdx.x;
  const unsigned run = u / per, rest = u - run * per;
  const int head = rest >> shift, eight = rest & ((1 << shift) - 1);
  const long long room = static_cast<long long>(p.width) << p.page_shift;
  int start = p.start ? p.start[b] : 0;
  long long length = p.lengths[b];
  if (start < 0 || length < 0 || length > room) {
    if (u == 0) set_bad_shape(status);
    length = start < 0 || length < 0 ? 0 : room;
    start = max(start, 0);
  }
  const long long at0 = static_cast<long long>(start & ~(kInt4Quad - 1)) + static_cast<long long>(run) * kInt4Quad;
  const int first = static_cast<int>(max(0ll, start - at0));
  const int last = static_cast<int>(
      min(static_cast<long long>(kInt4Quad), static_cast<long long>(start) + p.tokens - at0));  // of the rows written
  if (first >= last) return;
  const int held = static_cast<int>(max(0ll, min(static_cast<long long>(last), length - at0)));  // of those with a token
  int id = held > first ? p.table[b * p.table_ld + (at0 >> p.page_shift)] : -1;
  if (held > first && (id < 0 || id >= p.pages)) {
    set_bad_shape(status);
    id = -1;
  }
  const int in_page = static_cast<int>(at0 & ((1 << p.page_shift) - 1));
  const long long unit = static_cast<long long>(max(id, 0)) * p.kv_heads + head;
  T* out = static_cast<T*>(p.out[which]) + b * p.out_batch[which] + rest * 8 + (at0 - start) * p.out_ld[which];
  uint2 raw[kInt4Quad];
  uint32_t scale = 0;
  if (id >= 0) {  // (all four: the page holds them, written or not)
    if constexpr (INT4) {
      const uint8_t* codes = p.codes[which] + ((unit << p.page_shift) + in_page) * (p.dim / 2) + eight * 4;
#pragma unroll
      for (int j = 0; j < kInt4Quad; ++j) raw[j].x = *reinterpret_cast<const uint32_t*>(codes + j * (p.dim / 2));
      scale = *reinterpret_cast<const uint32_t*>(
          p.scales[which] + ((((unit << p.group_shift) + (eight >> 1)) << p.page_shift) + in_page));
    } else {
      const uint8_t* codes = p.codes[which] + ((unit << p.page_shift) + in_page) * p.dim + eight * 8;
#pragma unroll
      for (int j = 0; j < kInt4Quad; ++j) raw[j] = *reinterpret_cast<const uint2*>(codes + j * p.dim);
      scale = p.scales[which][unit];
    }
  }
#pragma unroll
  for (int j = 0; j < kInt4Quad; ++j) {
    if (j < first || j >= last) continue;
    T* to = out + j * p.out_ld[which];
    __align__(16) T value[8];
    if (id < 0 || j >= held) {
      const float zeros[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      store8<T>(value, zeros);
    } else if constexpr (INT4) {
      const uint32_t s = scale_pair(scale, scale_selector(j, j));
      uint32_t v[4];
      unpack4(raw[j].x, as_half2(s), minus72(s), v);
      const uint32_t ordered[4] = {__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                                   __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632)};
      store_half8<T>(value, ordered);
    } else {
      const float s = scale == 255 ? fp8_nan() : fp8_pow2(static_cast<int>(scale) - 127);
      float f[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t two = fp8_unpack2(((k < 2 ? raw[j].x : raw[j].y) >> (16 * (k & 1))) & 0xFFFFu);
        const float2 x = __half22float2(as_half2(two));
        f[2 * k] = x.x * s, f[2 * k + 1] = x.y * s;
      }
      store8<T>(value, f);
    }
    if (p.vec) {
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k)
        reinterpret_cast<uint4*>(to)[k] = reinterpret_cast<const uint4*>(value)[k];
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) to[c] = value[c];
    }
  }
}

int kv_read(cudaStream_t stream, bool int4, const ldb_kv_read_desc* desc) {
  if (const int rc = check_desc(desc, "kv_read")) return rc;
  const auto& [struct_size, dtype, cache, k, v, k_ld, k_batch, v_ld, v_batch, lengths, start, tokens] = *desc;
  const auto& [k_codes, v_codes, k_scales, v_scales, table, table_ld, pages, kv_heads, page, head_dim, width, batch] =
      cache;
  if (batch < 0 || tokens < 0) return fail(LDB_ERR_SHAPE, "kv_read: %d items of %d tokens", batch, tokens);
  if (dtype != LDB_F16 && dtype != LDB_F32 && dtype != LDB_BF16)
    return fail(LDB_ERR_INVALID, "kv_read: unknown element type %d", dtype);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(LDB_ERR_SHAPE, "kv_read: head_dim %d (32, 64 or 128)", head_dim);
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return fail(LDB_ERR_SHAPE, "kv_read: pages of %d tokens (16, 32, 64 or 128)", page);
  if (pages <= 0 || kv_heads <= 0 || width <= 0 || table_ld < width)
    return fail(LDB_ERR_SHAPE, "kv_read: %d pages, %d heads, table of %d", pages, kv_heads, width);
  if (batch == 0 || tokens == 0) return LDB_OK;
  if (!k || !v || !k_codes || !v_codes || !k_scales || !v_scales || !table || !lengths)
    return fail(LDB_ERR_INVALID, "kv_read: null pointer");
  const long long row = static_cast<long long>(kv_heads) * head_dim;
  const long long units = ((static_cast<long long>(tokens) + kInt4Quad - 2) / kInt4Quad + 1) * (row / 8);
  if ((tokens > 1 && (k_ld < row || v_ld < row)) || (batch > 1 && (k_batch < row || v_batch < row)) || batch > 65535 ||
      units > 0x7FFFFF00ll)
    return fail(LDB_ERR_SHAPE, "kv_read: row or item strides below %lld, more than 65535 items, or %lld channels and "
                "tokens", row, units);
  for (const uint8_t* t : {k_codes, v_codes})
    if (reinterpret_cast<uintptr_t>(t) % 16) return fail(LDB_ERR_ALIGNMENT, "kv_read: codes must be 16-byte aligned");
  if (int4 && (reinterpret_cast<uintptr_t>(k_scales) % 16 || reinterpret_cast<uintptr_t>(v_scales) % 16))
    return fail(LDB_ERR_ALIGNMENT, "kv_read: scales must be 16-byte aligned");
  unsigned int* status = device_status_ptr();
  if (!status) return fail(LDB_ERR_CUDA, "kv_read: no device status word");
  ReadParams p{};
  p.codes[0] = k_codes, p.codes[1] = v_codes, p.scales[0] = k_scales, p.scales[1] = v_scales;
  p.out[0] = k, p.out[1] = v, p.out_ld[0] = k_ld, p.out_ld[1] = v_ld, p.out_batch[0] = k_batch, p.out_batch[1] = v_batch;
  p.table = table, p.table_ld = table_ld, p.lengths = lengths, p.start = start;
  p.pages = pages, p.kv_heads = kv_heads, p.width = width, p.dim = head_dim, p.tokens = tokens;
  p.page_shift = page == 16 ? 4 : (page == 32 ? 5 : (page == 64 ? 6 : 7));
  p.group_shift = head_dim == 32 ? 1 : (head_dim == 64 ? 2 : 3);
  const int es = dtype == LDB_F32 ? 4 : 2;
  p.vec = 1;
  for (int i = 0; i < 2; ++i)
    if (reinterpret_cast<uintptr_t>(p.out[i]) % 16 || p.out_ld[i] * es % 16 || p.out_batch[i] * es % 16) p.vec = 0;
  const dim3 grid(static_cast<unsigned>((units + kThreads - 1) / kThreads), batch, 2);
  auto run = [&](auto kernel4, auto kernel8) {
    return launch_kernel(int4 ? kernel4 : kernel8, grid, dim3(kThreads), 0, stream, "kv_read launch", p, status);
  };
  if (dtype == LDB_F16) return run(kv_read_kernel<__half, true>, kv_read_kernel<__half, false>);
  if (dtype == LDB_BF16) return run(kv_read_kernel<__nv_bfloat16, true>, kv_read_kernel<__nv_bfloat16, false>);
  return run(kv_read_kernel<float, true>, kv_read_kernel<float, false>);
}

}  // namespace
}  // namespace ldb

extern "C" {

int ldb_kv_read_fp8(cudaStream_t stream, const ldb_kv_read_desc* desc) { return ldb::kv_read(stream, false, desc); }

int ldb_kv_read_int4(cudaStream_t stream, const ldb_kv_read_desc* desc) { return ldb::kv_read(stream, true, desc); }

}  // extern "C"
