"""Cache attention where an item's tokens are cut into ranges that a second kernel joins.

The bounds are those of the cache's other tests: the ranges' partial rows are
FP32 and add 2^-22 relative, inside their 2^-18."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_cache as oracle
from tests.test_kv_cache_gpu import check_attention, host, ints, make_cache, make_table

pytestmark = pytest.mark.gpu


def token_ranges(batch, queries, heads, kv_heads, dim, capacity):
    """Ranges that the many-row kernel cuts a table of this capacity into: from the size of the partial rows."""
    need = ctypes.c_size_t()
    _lib.call("ldb_kv_attention_fp8_table_workspace_size", batch, queries, heads, kv_heads, dim, capacity,
              ctypes.byref(need))
    return need.value // (batch * heads * queries * (dim + 2) * 4)


def without_nan(ref):
    return {name: x.nan_to_num(0.0) for name, x in ref.items()}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,queries,heads,group,dim,page,width", [
    ([1100, 0, 130], 50, 1, 1, 64, 64, 20), ([2000], 99, 1, 3, 128, 128, 16), ([700, 1500], 33, 2, 2, 32, 16, 100),
    ([5], 61, 1, 1, 128, 64, 40)])
def test_many_rows_over_ranges(cuda_device, dtype, causal, lengths, queries, heads, group, dim, page, width):
    """Rows that end inside a warp, ranges without tokens, and NaN values that all, some or none of the rows see."""
    batch = len(lengths)
    assert token_ranges(batch, queries, heads * group, heads, dim, width * page) > 1
    table, pages = make_table(batch, width, cuda_device, 11)
    cache = make_cache(pages, heads, dim, page, cuda_device, 12)
    n = lengths[0]
    for tok, channel in ((n - 1, 3), (n // 2, 9), (max(0, n - queries // 2), dim - 1)):
        cache.v.view(torch.uint8)[int(table[0, tok // page]), heads - 1, tok % page, channel] = 0x7F
    q = torch.randn(batch, queries, heads * group * dim, generator=torch.Generator().manual_seed(13)).to(dtype)
    args = (q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device))
    got = kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal)
    ref = oracle.attention(q, *host(cache), table, lengths, group, dim ** -0.5, causal)
    nan = torch.isnan(ref["out"])
    assert nan.any() and torch.equal(torch.isnan(got.cpu().view(nan.shape)), nan)
    check_attention(torch.where(nan.to(cuda_device), 0.0, got.view(nan.shape)), without_nan(ref), dtype)
    assert torch.equal(kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal).nan_to_num(7.0),
                       got.nan_to_num(7.0))
    assert _lib.device_status(reset=True) == 0
