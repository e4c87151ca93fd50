// The many-row kernel of the 4-bit cache's attention (p's shapes and pointers filled in), and the
// bytes of the partial rows of its ranges for a table of `capacity` tokens.
#pragma once

#include "kv_attention.cuh"

namespace ldb {

size_t kv_int4_tile_workspace(int batch, int kv_heads, long long rows, int head_dim, long long capacity);
int kv_int4_attention_tiles(cudaStream_t stream, KvTileParams p, int head_dim, int dtype, float scale, void* workspace,
                            unsigned int* status);

}  // namespace ldb
