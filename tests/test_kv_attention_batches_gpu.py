"""Cache attention of few rows where its line of tiles is cut in the ways that small calls do not reach:
more pairs of item and head than warps, lengths scanned in several rounds, and pairs of more parts
than a block of the joining kernel has threads."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_cache as oracle
from tests.test_kv_attention_precision_gpu import attend, check, inputs
from tests.test_kv_cache_gpu import check_attention, host, ints, make_cache, make_table

pytestmark = pytest.mark.gpu


def warps(dim):
    """Of the few-row kernel's grid: four to a block, two blocks an SM at 128 channels, else three."""
    return torch.cuda.get_device_properties(0).multi_processor_count * 4 * (2 if dim == 128 else 3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,queries,heads,group,dim,page,most,causal", [
    (300, 1, 8, 2, 32, 16, 70, False), (300, 1, 8, 4, 128, 64, 130, True), (257, 3, 8, 1, 64, 32, 100, True),
    (600, 5, 3, 2, 64, 16, 40, True), (2048, 1, 1, 1, 32, 16, 33, False)])
def test_more_pairs_than_warps(cuda_device, dtype, batch, queries, heads, group, dim, page, most, causal):
    """Ragged items, idle ones among them (the first, the last and runs of them)."""
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(1, most + 1, (batch,), generator=g)
    lengths[torch.rand(batch, generator=g) < 0.15] = 0
    lengths[0], lengths[-1], lengths[120:135] = 0, 0, 0
    lengths = lengths.tolist()
    assert batch * heads > warps(dim)
    table, pages = make_table(batch, -(-most // page), cuda_device, 3)
    cache = make_cache(pages, heads, dim, page, cuda_device, 4)
    q = torch.randn(batch, queries, heads * group * dim, generator=g).to(dtype)
    args = (q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device))
    got = kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal)
    check_attention(got, oracle.attention(q, *host(cache), table, lengths, group, dim ** -0.5, causal), dtype)
    assert torch.equal(kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal), got)
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,tokens,queries,dim,page", [
    (1, 40000, 1, 128, 64), (1, 60001, 3, 64, 128), (8, 20000, 1, 128, 64), (2, 30017, 20, 32, 16)])
def test_pairs_of_many_parts(cuda_device, dtype, heads, tokens, queries, dim, page):
    """From 64 to over 1024 parts of a pair: the joining kernel's rounds over its threads."""
    assert min(warps(dim) // heads, tokens // 32) >= 64
    q, k, v = inputs(heads, tokens, queries, dim, dtype, heads + tokens)
    used = -(-tokens // page)
    exps = [-7] * used, [(-9, -6, -8, -7)[i % 4] for i in range(used)]
    got = attend(q, k, v, *exps, page, dim ** -0.5)
    check(got, q, k, v, *exps, page, dim ** -0.5)
