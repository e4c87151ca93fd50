// Layout of the paged 8-bit key/value cache and the operand checks that its
// kernels share.  codes[page][kv head][token in page][channel] (e4m3), scales
// [page][kv head] (E8M0); an item's tokens lie in the pages of its table row.
#pragma once

#include "fp8.cuh"

namespace ldb {

constexpr int kKvMaxExponent = 96;  // page scales stay within 2^-96 .. 2^96: so do the terms of a softmax sum that count

struct KvView {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  const int* table;    // [batch][table_ld], `width` entries used
  const int* lengths;  // [batch]
  long long table_ld;
  int pages, kv_heads, page, width, batch;
};

// Tokens of item b: a length outside [0, width * page] is cut and reported.
__device__ __forceinline__ int kv_length(const KvView& c, int b, unsigned int* status) {
  const int n = c.lengths[b];
  const long long room = static_cast<long long>(c.width) * c.page;
  if (n >= 0 && n <= room) return n;
  set_bad_shape(status);
  return n < 0 ? 0 : static_cast<int>(room);
}

}  // namespace ldb
