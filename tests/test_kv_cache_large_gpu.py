"""A cache whose codes pass 2^32 bytes: writing to its last pages and reading them."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_cache as oracle
from tests.test_kv_cache_gpu import check_attention, host, ints, same_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("queries", [1, 20, 70])
def test_pages_past_32_bits(cuda_device, queries):
    heads, dim, page, tokens = 8, 128, 128, 300
    pages = 2 ** 32 // (heads * dim * page) + 9
    cache = kv_cache.KvCacheFp8.empty(pages, heads, dim, page=page, device=cuda_device)
    assert cache.k.numel() > 2 ** 32
    used = [pages - 1, 0, pages - 6, pages - 3]
    table = torch.tensor([used], dtype=torch.int32)
    g = torch.Generator().manual_seed(queries)
    k, v = (torch.randn(1, tokens, heads * dim, generator=g).to(torch.bfloat16) for _ in range(2))
    for t in (cache.k, cache.v):
        t.view(torch.uint8)[used] = 0
    for t in (cache.k_scale, cache.v_scale):
        t.view(torch.uint8)[used] = 127
    start = ints([0], cuda_device)
    kv_cache.kv_append(cache, k[:, :200].to(cuda_device), v[:, :200].to(cuda_device), table.to(cuda_device), start)
    kv_cache.kv_append(cache, k[:, 200:].to(cuda_device), v[:, 200:].to(cuda_device), table.to(cuda_device), start + 200)
    small = kv_cache.KvCacheFp8(*(t.view(torch.uint8)[used].view(t.dtype) for t in cache))
    near = torch.arange(len(used), dtype=torch.int32)[None]
    want = [torch.zeros_like(t) for t in host(small)]
    for (codes, e), new in zip(((want[0], want[1]), (want[2], want[3])), (k, v)):
        rows = new.view(1, tokens, heads, dim)
        oracle.append(codes, e, rows[:, :200], near, [0], [200])
        oracle.append(codes, e, rows[:, 200:], near, [200], [tokens - 200])
    same_cache(small, want)
    q = torch.randn(1, queries, heads * dim, generator=g).to(torch.bfloat16)
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints([tokens], cuda_device),
                                scale=dim ** -0.5, causal=True)
    check_attention(got, oracle.attention(q, *want, near, [tokens], 1, dim ** -0.5, True), torch.bfloat16)
    assert _lib.device_status(reset=True) == 0
