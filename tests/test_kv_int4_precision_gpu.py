"""4-bit cache attention where weights span many powers of two, and references grow late.

Output bound, per value: a weight (in units of the row's largest) is rounded to f16 once, 2^-11 relative, or half
of f16's least step, 2^-25, where it is subnormal; the largest weighs at least 2^11 for up to 48 rows of a
key/value head and 2^7 from 49 on, so that is 2^-36 and 2^-32 of the largest.  A score is off by its FP32 sum, 8 * 2^-23 of its
terms' magnitudes; a weight moves by that much relative, once itself and once in the sum.  Exponential,
sum and division add 2^-18, and the output is rounded once."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_int4 as oracle
from tests.test_kv_int4_gpu import TINY, UNIT, ints, make_table

pytestmark = pytest.mark.gpu

MANY_ROWS = 49  # of one key/value head: from here on the many-row kernel runs
HEADROOM = {False: 11, True: 7}
BLOCK = 128  # tokens that either kernel takes at a time, or several times those


def attend(q, codes, scales, page, scale, items):
    """(items, L, heads * dim) outputs over the same (heads, tokens, dim) codes and (heads, tokens, dim / 16) scale bytes of
    keys and values for each item, which share its pages."""
    heads, tokens, dim = codes[0].shape
    used = -(-tokens // page)
    table, pages = make_table(1, used, 3)
    tensors = []
    for c in codes:
        t = torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8)
        for slot in range(used):
            part = c[:, slot * page: (slot + 1) * page]
            t[int(table[0, slot]), :, : part.shape[1]] = part[..., ::2] | (part[..., 1::2] << 4)
        tensors.append(t)
    for s in scales:
        t = torch.full((pages, heads, dim // 16, page), oracle.NAN, dtype=torch.uint8)  # (nobody sees these)
        for slot in range(used):
            part = s[:, slot * page: (slot + 1) * page]
            t[int(table[0, slot]), ..., : part.shape[1]] = part.transpose(1, 2)
        tensors.append(t)
    cache = kv_cache.KvCacheInt4(*(t.cuda() for t in tensors))
    args = (q.repeat(items, 1, 1).cuda(), cache, table.repeat(items, 1).cuda(), ints([tokens] * items, "cuda"))
    got = kv_cache.kv_attention(*args, scale=scale)
    assert torch.equal(got, kv_cache.kv_attention(*args, scale=scale))
    assert _lib.device_status(reset=True) == 0
    return got.cpu()


def values_of(codes, scales):
    table = torch.tensor(oracle.SCALES, dtype=torch.float64)
    return (codes.double() - 8) * table[scales.long()].repeat_interleave(16, -1)


def check(got, q, codes, scales, scale, sharp):
    """``sharp``: the groups of channels where the bound has to lie below 2^-5 of the mean output."""
    k, v = (values_of(c, s) for c, s in zip(codes, scales))
    heads, tokens, dim = k.shape
    queries, dtype = q.shape[1], q.dtype
    rows = q.double().view(queries, -1, dim)
    group = rows.shape[1] // heads
    headroom = HEADROOM[queries * group >= MANY_ROWS]
    for h in range(rows.shape[1]):
        keys, values = k[h // group], v[h // group]
        w = torch.softmax(rows[:, h] @ keys.T * scale, -1)
        off = 8 * 2.0 ** -23 * (rows[:, h].abs() @ keys.abs().T).amax(-1, keepdim=True) * abs(scale)
        delta = torch.maximum(2.0 ** -11 * w, 2.0 ** -(25 + headroom) * w.amax(-1, keepdim=True))
        delta = delta + w * (2.0 ** -18 + 2 * off)
        out, bound = w @ values, delta @ values.abs()
        for n in sharp:
            at = slice(16 * n, 16 * (n + 1))
            assert (bound[:, at].mean(-1) <= 2.0 ** -5 * out[:, at].abs().mean(-1)).all(), "the case says nothing"
        bound = bound + UNIT[dtype] * out.abs() * (1 + 2.0 ** -8) + TINY[dtype]
        err = (got.double().view(got.shape[0], queries, -1, dim)[:, :, h] - out).abs()
        assert (err <= bound).all(), float((err / bound).max())


def inputs(heads, tokens, queries, group, dim, dtype, seed):
    """Queries and random keys that leave out the keys' first group of channels, whose channel 0 the caller sets under the
    queries' one (1); positive values."""
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(low, 16, (heads, tokens, dim), generator=g, dtype=torch.uint8) for low in (0, 9)]
    scales = [torch.full((heads, tokens, dim // 16), 112, dtype=torch.uint8) for _ in range(2)]  # 0.5
    codes[0][..., :16], scales[0][..., 0] = 8, 120  # 1.0
    q = 0.5 * torch.randn(1, queries, heads * group, dim, generator=g)
    q[..., 0] = 1.0
    return q.flatten(2).to(dtype), codes, scales


# queries, group, dim, page, items: one range an item where there are many; from 49 rows on one tile whose blocks alternate where 40
# items of two key/value heads and this many tokens are there, two tiles, and several ranges of tokens
SHAPES = [(1, 1, 128, 64, 900), (1, 4, 64, 16, 1), (4, 4, 32, 32, 300), (3, 16, 128, 128, 1), (16, 1, 64, 64, 1),
          (60, 1, 128, 64, 80), (30, 2, 64, 16, 80), (60, 1, 32, 128, 80), (60, 1, 128, 128, 1), (300, 1, 128, 64, 80),
          (150, 2, 64, 16, 1), (300, 1, 32, 32, 2)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rise", [9.0, 10.0, -10.0])
@pytest.mark.parametrize("queries,group,dim,page,items", SHAPES)
def test_scores_that_rise_block_by_block(cuda_device, dtype, rise, queries, group, dim, page, items):
    """Blocks' scores 2^9 or 2^10 above those before (or below): the reference grows with each while the output is not zero.
    Each group of channels has values in one block alone, the first group in that of the largest weights, and so on."""
    blocks = 8
    tokens = 4 * BLOCK * blocks
    q, codes, scales = inputs(2, tokens, queries, group, dim, dtype, queries + dim)
    level = torch.arange(tokens) // (4 * BLOCK)  # (runs of four blocks: ranges and tiles grow within, too)
    codes[0][..., 0], scales[0][..., 0] = 9, (120 + level).to(torch.uint8)  # 1 + level / 8
    scale = abs(rise) * 8 / 1.4426950408889634
    q = (q.float() / (scale * dim ** 0.5)).view(1, queries, -1, dim)  # (the rest of the scores spread by a few units)
    q[..., 0] = 1.0 if rise > 0 else -1.0
    q = q.flatten(2).to(dtype)
    for n in range(dim // 16):
        held = blocks - 1 - n if rise > 0 else n
        codes[1][..., 16 * n: 16 * (n + 1)][:, level != held] = 8
    got = attend(q, codes, scales, page, scale, items)
    sharp = [n for n in range(dim // 16) if abs(rise) * n <= (10 if queries * group >= MANY_ROWS else 20)]
    check(got, q, codes, scales, scale, sharp)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("place", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("queries,group,dim,page,items", SHAPES)
def test_a_key_that_takes_nearly_all_the_weight(cuda_device, dtype, place, queries, group, dim, page, items):
    """One token takes most of the weight and its values are zero: the output is the rest's."""
    tokens = 3300
    q, codes, scales = inputs(2, tokens, queries, group, dim, dtype, queries + dim)
    scale, at = dim ** -0.5, int(place * (tokens - 1))
    codes[1][:, at] = 8
    codes[0][:, at] = 8
    codes[0][:, at, 0], scales[0][:, at, 0] = 12, 152  # 4 * 16
    q = q.view(1, queries, -1, dim)
    q[..., 0] = 15.0 / (64 * scale)
    got = attend(q.flatten(2), codes, scales, page, scale, items)
    check(got, q.flatten(2), codes, scales, scale, range(dim // 16))
