"""4-bit cache attention where scores lie far past 2^20, at either sign.

Each query has one channel that is not zero, so a score is exact and its row's keys are either equal or so
far apart (2^-4 of the largest, and never less than 2^7 as a power of two) that the definition gives the
keys of the largest score equal weights and the others none.  So must the kernels: rounding a score moves
equal ones alike.  What remains is the weights' 2^-11, the sums' 2^-18 and the output's own rounding."""

from __future__ import annotations

import math

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_int4 as oracle
from tests.test_kv_int4_gpu import TINY, UNIT, check_attention, host, ints, make_cache, make_table

pytestmark = pytest.mark.gpu

SHAPES = [  # lengths, queries, kv heads, group, dim, page, causal
    ([300, 0, 5, 64], 1, 2, 4, 128, 64, False), ([700, 33], 3, 2, 5, 64, 16, True), ([2100], 4, 1, 12, 32, 128, True),
    ([5000], 1, 1, 1, 128, 128, False), ([300, 129], 60, 2, 1, 128, 64, True), ([700], 300, 1, 1, 64, 16, True),
    ([3000], 130, 1, 2, 32, 128, False), ([3200, 2000] + [5] * 35, 60, 4, 1, 128, 64, False),
    ([3200, 2000] + [5] * 35, 32, 4, 4, 32, 128, True)]
# Order of the keys: all the same, by chance, and in order, so that the largest score grows all the way or never.
KEYS = ("equal", "chance", "rising", "falling")


def inputs(lengths, queries, heads, group, dim, page, keys, sign, dtype, device):
    """A cache whose keys are a code of channel 5 under one scale (1), and queries of that channel alone."""
    table, pages = make_table(len(lengths), -(-max(lengths) // page) + 1, 11)
    cache = make_cache(pages, heads, dim, page, device, 12, 96, 112)
    g = torch.Generator().manual_seed(13)
    tokens = table.shape[1] * page
    codes = {"equal": torch.full((tokens,), 13), "chance": torch.randint(1, 16, (tokens,), generator=g),
             "rising": 1 + torch.arange(tokens) * 14 // max(lengths),
             "falling": 15 - torch.arange(tokens) * 14 // max(lengths)}[keys].clamp(1, 15)
    if sign < 0:
        codes = codes.clamp(max=7)  # (negative keys alone, or zero where every score of a row is to be zero)
    k = torch.full((pages, heads, page, dim), 8, dtype=torch.uint8)
    for b in range(len(lengths)):
        for slot in range(table.shape[1]):
            k[int(table[b, slot]), :, :, 5] = codes[slot * page: (slot + 1) * page].to(torch.uint8)
    cache.k.copy_(k[..., ::2] | (k[..., 1::2] << 4))
    cache.k_scale.fill_(120)  # 1.0
    q = torch.zeros(len(lengths), queries, heads * group, dim)
    q[..., 5] = 1 + torch.rand(q.shape[:-1], generator=g)
    if sign == 0:
        q[..., 5] *= torch.randint(0, 2, q.shape[:-1], generator=g) * 2 - 1
    return cache, table, q.flatten(2).to(dtype)


def definition(q, cache, table, lengths, group, scale, causal):
    """Outputs (B, L, heads * group, dim) and the weighted magnitudes of their values, item by item."""
    codes_k, codes_v, scales_k, scales_v = host(cache)
    k, v = oracle.values(codes_k, scales_k), oracle.values(codes_v, scales_v)
    heads, dim = k.shape[1], k.shape[3]
    batch, m = q.shape[:2]
    q = q.double().view(batch, m, heads, group, dim).permute(0, 2, 3, 1, 4)
    out, size = (torch.zeros(batch, heads, group, m, dim, dtype=torch.float64) for _ in range(2))
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        keys, values = (oracle.rows(x, table, b, n)[:, None] for x in (k, v))
        scores = q[b] @ keys.transpose(-1, -2) * scale
        seen = torch.full((m,), n) if not causal else n - m + 1 + torch.arange(m)
        scores = scores.masked_fill(torch.arange(n) >= seen[:, None], -math.inf)
        p = torch.softmax(scores, -1).nan_to_num(0.0)  # (rows that see nothing)
        out[b], size[b] = p @ values, p @ values.abs()
    return [x.permute(0, 3, 1, 2, 4).flatten(2, 3) for x in (out, size)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("keys", KEYS)
@pytest.mark.parametrize("sign", [0, -1])
@pytest.mark.parametrize("lengths,queries,heads,group,dim,page,causal", SHAPES)
def test_scores_far_past_their_rounding(cuda_device, dtype, keys, sign, lengths, queries, heads, group, dim, page, causal):
    cache, table, q = inputs(lengths, queries, heads, group, dim, page, keys, sign, dtype, cuda_device)
    args = (q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device))
    out, size = definition(q, cache, table, lengths, group, 2.0 ** 20, causal)  # (one for all: only ties have any weight)
    bound = (2.0 ** -11 + 2.0 ** -18) * size + UNIT[dtype] * out.abs() * (1 + 2.0 ** -8) + TINY[dtype]
    for power in (12, 19, 20, 21, 22, 24, 25, 27, 30, 40, 64, 99, 118):
        got = kv_cache.kv_attention(*args, scale=math.ldexp(1.0, power), causal=causal)
        bad = ~((got.cpu().double().view(out.shape) - out).abs() <= bound)
        assert not bad.any(), (power, int(bad.sum()), int((~torch.isfinite(got)).sum()))
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lost", [False, True])
@pytest.mark.parametrize("lengths,queries,heads,group,dim,page,causal", [
    ([300, 0, 5, 64], 7, 2, 1, 128, 64, True), ([700, 33], 3, 2, 5, 64, 16, False), ([2100], 4, 1, 12, 32, 128, True),
    ([300, 129], 60, 2, 1, 128, 64, True), ([700], 300, 1, 1, 64, 16, False), ([3000], 130, 1, 2, 32, 128, True),
    ([3200, 2000] + [5] * 35, 60, 4, 1, 128, 64, True), ([3200, 2000] + [5] * 35, 32, 4, 4, 32, 128, False)])
def test_rows_beside_far_ones(cuda_device, dtype, lost, lengths, queries, heads, group, dim, page, causal):
    """Every third query's scores are about 2^25, one query is NaN and one has an infinity: the others' outputs are theirs."""
    if lost and causal:
        pytest.skip("a query's place among the tokens would be another")
    table, pages = make_table(len(lengths), -(-max(lengths) // page) + 1, 11)
    cache = make_cache(pages, heads, dim, page, cuda_device, 12, 96, 112)
    q = torch.randn(len(lengths), queries, heads * group * dim, generator=torch.Generator().manual_seed(13))
    scale = 2.0 ** 14 * dim ** -0.5
    q *= 2.0 ** -13
    q[:, ::3] *= 2.0 ** 20
    q[0, -2, 3], q[0, -1, 0] = float("nan"), float("inf")
    q = q.to(dtype)
    seen, kept = lengths, table
    if lost:  # the first item's second page
        kept = table.clone()
        kept[0, 1:-1] = table[0, 2:]
        seen = [lengths[0] - page, *lengths[1:]]
        table = table.clone()
        table[0, 1] = pages
    got = kv_cache.kv_attention(q.to(cuda_device), cache, table.to(cuda_device), ints(lengths, cuda_device), scale=scale,
                                causal=causal).cpu()
    assert _lib.device_status(reset=True) == (2 if lost else 0)
    heads_of = got.view(len(lengths), queries, -1, dim)
    assert torch.isnan(heads_of[0, -2, 0]).all() and torch.isnan(heads_of[0, -1, 0]).all()
    far = [i for i in range(0, queries, 3) if i < queries - 2]
    codes_k, codes_v, scales_k, scales_v = host(cache)
    v = oracle.values(codes_v, scales_v)
    assert (got[:, far].abs().double() <= v.abs().max() * (1 + 2.0 ** -7)).all()
    rest = [i for i in range(queries) if i % 3 and i < queries - 2]
    ref = oracle.attention(q, oracle.values(codes_k, scales_k), v, kept, seen, group, scale, causal)
    check_attention(got[:, rest], {k: x[:, rest] for k, x in ref.items()}, dtype)
