"""4-bit cache attention of few rows with more pairs (of an item, a key/value head and a tile of rows) than the grid has
warps: ranges that hold several whole pairs, and pairs cut by a range's end."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from tests.test_kv_int4_gpu import check_attention, ints, make_cache, reference

pytestmark = pytest.mark.gpu


def warps(dim, rows):
    """Of the few-row kernel's grid: four a block, three blocks an SM or two."""
    blocks = 2 if dim == 128 and rows > 8 else 3
    return 4 * blocks * torch.cuda.get_device_properties(0).multi_processor_count


def ragged(batch, most, long):
    lengths = [(37 * i) % most for i in range(batch)]  # (some of them idle)
    for at, n in long.items():
        lengths[at] = n
    return lengths


@pytest.mark.parametrize("lengths,queries,heads,group,dim,page,causal,dtype", [
    (ragged(300, 90, {5: 3000, 299: 1700}), 1, 8, 1, 128, 64, True, torch.bfloat16),
    (ragged(300, 70, {0: 2500}), 1, 8, 1, 32, 16, False, torch.float16),
    (ragged(257, 90, {100: 1500, 101: 900}), 3, 8, 1, 64, 32, True, torch.float16),
    (ragged(2048, 40, {1000: 4000}), 1, 1, 4, 64, 64, False, torch.bfloat16),
    (ragged(150, 90, {7: 2100}), 5, 8, 4, 64, 128, True, torch.bfloat16),
    (ragged(80, 120, {79: 2500, 40: 600}), 8, 8, 6, 128, 64, False, torch.float16),
    (ragged(120, 60, {50: 3100}), 16, 8, 2, 32, 32, True, torch.float16)])
def test_more_pairs_than_warps(cuda_device, lengths, queries, heads, group, dim, page, causal, dtype):
    batch, rows = len(lengths), queries * group
    tiles = -(-rows // (8 if rows <= 8 else 16))
    assert rows < 49 and batch * heads * tiles > warps(dim, rows)
    table = torch.full((batch, -(-max(lengths) // page)), -1, dtype=torch.int32)
    used = [-(-n // page) for n in lengths]
    order, at = torch.randperm(sum(used), generator=torch.Generator().manual_seed(5)).to(torch.int32), 0
    for b, n in enumerate(used):
        table[b, :n] = order[at: at + n]
        at += n
    cache = make_cache(at, heads, dim, page, cuda_device, 6, 96, 112)
    q = torch.randn(batch, queries, heads * group * dim, generator=torch.Generator().manual_seed(8)).to(dtype)
    args = (q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device))
    out = torch.full_like(args[0], 7.0)
    got = kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal, out=out)
    check_attention(got, reference(q, cache, table, lengths, group, dim ** -0.5, causal), dtype)
    assert torch.equal(kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal), got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = kv_cache.kv_attention(*args, scale=dim ** -0.5, causal=causal)
    again.fill_(7.0)
    graph.replay()
    assert torch.equal(again, got) and _lib.device_status(reset=True) == 0
