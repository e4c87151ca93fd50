"""Cache attention where the weights of the value product span many powers of two.

Output bound, per value: a weight p 2^ev (in units of the row's largest) is
rounded to f16 with a headroom, 2^15 for few rows and 2^7 for many: 2^-11
relative, or 2^-25 of the largest over the headroom where it is subnormal.  A score is off by its
FP32 sum, 8 * 2^-23 of its terms' magnitudes, and by what the queries' e4m3 parts
leave, 2^-18 of the row's largest channel times the key's magnitudes; a weight
moves by that much relative, once itself and once in the sum.  Exponential, sum and division add
2^-18, and the output is rounded once.  Every case also shows that this bound
lies below 2^-5 of the output."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from lesiondiffusion_mlx_b200.fp8 import CODES, SCALES
from tests.test_kv_cache_gpu import TINY, UNIT, ints, make_table

pytestmark = pytest.mark.gpu

MANY_ROWS = 49  # of one key/value head: from here on the many-row kernel runs
HEADROOM = {False: 15, True: 7}


def attend(q, k, v, k_exp, v_exp, page, scale, *, width=None, items=1):
    """(B, L, heads, dim) outputs of ``kv_attention`` over the same (heads, tokens, dim) code values for each item."""
    heads, tokens, dim = k.shape
    used = -(-tokens // page)
    table, pages = make_table(1, width or used, "cpu", 3)
    codes = [torch.zeros(pages, heads, page, dim) for _ in range(2)]
    scales = [torch.full((pages, heads), 127, dtype=torch.uint8) for _ in range(2)]
    for slot in range(used):
        at, n = int(table[0, slot]), min(page, tokens - slot * page)
        for c, s, x, e in ((codes[0], scales[0], k, k_exp), (codes[1], scales[1], v, v_exp)):
            c[at, :, :n] = x[:, slot * page : slot * page + n]
            s[at] = e[slot] + 127
    cache = kv_cache.KvCacheFp8(*(c.to(CODES).cuda() for c in codes), *(s.view(SCALES).cuda() for s in scales))
    args = (q.repeat(items, 1, 1).cuda(), cache, table.repeat(items, 1).cuda(), ints([tokens] * items, "cuda"))
    got = kv_cache.kv_attention(*args, scale=scale)
    assert torch.equal(got, kv_cache.kv_attention(*args, scale=scale))
    assert _lib.device_status(reset=True) == 0
    return got.cpu()


def check(got, q, k, v, k_exp, v_exp, page, scale):
    heads, tokens, dim = k.shape
    queries, dtype = q.shape[1], q.dtype
    exps = [torch.exp2(torch.tensor(e, dtype=torch.float64)).repeat_interleave(page)[:tokens] for e in (k_exp, v_exp)]
    headroom = HEADROOM[queries * q.shape[2] // (heads * dim) >= MANY_ROWS]
    rows = q.double().view(queries, heads, dim)
    for h in range(heads):
        keys = k[h].double() * exps[0][:, None]
        p = torch.softmax(rows[:, h] @ keys.T * scale, -1)
        off = (8 * 2.0 ** -23 * (rows[:, h].abs() @ keys.abs().T)
               + 2.0 ** -18 * rows[:, h].abs().amax(-1, keepdim=True) * keys.abs().sum(-1)) * abs(scale)
        w = p * exps[1]
        delta = torch.maximum(2.0 ** -11 * w, 2.0 ** -(25 + headroom) * w.amax(-1, keepdim=True))
        delta = delta + w * (2.0 ** -18 + 2 * off.amax(-1, keepdim=True))
        out = w @ v[h].double()
        bound = delta @ v[h].double().abs()
        assert (bound <= 2.0 ** -5 * out.abs()).all(), "the case says nothing"
        bound = bound + UNIT[dtype] * out.abs() * (1 + 2.0 ** -8) + TINY[dtype]
        err = (got.double().view(got.shape[0], queries, heads, dim)[:, :, h] - out).abs()
        assert (err <= bound).all(), float((err / bound).max())


def inputs(heads, tokens, queries, dim, dtype, seed):
    """Queries, keys whose scores without channel 0 spread by about one, and positive values."""
    g = torch.Generator().manual_seed(seed)
    k = (60 * torch.randn(heads, tokens, dim, generator=g)).clamp(-448, 448).to(CODES).float()
    v = (60 * torch.randn(heads, tokens, dim, generator=g)).abs().clamp(1, 448).to(CODES).float()
    k[:, :, 0] = 0
    q = torch.randn(1, queries, heads * dim, generator=g)
    return q.to(dtype), k, v


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,queries,dim,page,items,nats", [
    (8192, 1, 128, 64, 1, 18.0), (4000, 1, 128, 64, 700, 17.0), (1000, 7, 64, 16, 900, 15.0), (300, 14, 32, 32, 900, 13.0),
    (1500, 60, 128, 64, 80, 17.0), (1000, 200, 64, 16, 80, 17.0), (500, 300, 32, 128, 40, 16.0)])
def test_a_key_that_takes_nearly_all_the_weight(cuda_device, dtype, tokens, queries, dim, page, items, nats):
    """The first token takes up to 0.9998 of the weight and its values are zero: the output is the rest's.
    (Many items: each is one range of tokens, whose reference the first token sets.)"""
    q, k, v = inputs(2, tokens, queries, dim, dtype, tokens + queries)
    scale, pages = dim ** -0.5, -(-tokens // page)
    k[:, 0], v[:, 0] = 0, 0
    k[:, 0, 0] = 320  # times 2^-6: 5
    q.view(queries, 2, dim)[..., 0] = nats / (5 * scale)
    exps = [-6] * pages, [-2] * pages
    got = attend(q, k, v, *exps, page, scale, items=items)
    check(got, q, k, v, *exps, page, scale)


@pytest.mark.parametrize("queries,dim,page,items", [(1, 128, 64, 700), (12, 64, 16, 900), (2, 64, 16, 1), (60, 128, 128, 1),
                                                    (150, 32, 32, 1), (60, 64, 64, 100)])
@pytest.mark.parametrize("zero_page", [0, 2])
def test_a_page_of_zero_values(cuda_device, queries, dim, page, items, zero_page):
    """Zero values have the scale 1, which dwarfs the scales of small ones beside them."""
    tokens = 5 * page - 3
    q, k, v = inputs(2, tokens, queries, dim, torch.bfloat16, queries)
    v[:, zero_page * page : (zero_page + 1) * page] = 0
    v_exp = [-18, -16, -22, -20, -17]
    v_exp[zero_page] = 0
    exps = [-7] * 5, v_exp
    got = attend(q, k, v, *exps, page, dim ** -0.5, items=items)
    check(got, q, k, v, *exps, page, dim ** -0.5)


SPREADS = [[96, -96, 96, -96, -96], [-96, -96, 96, -20, 3], [96, -96, -60, -30, -10], [-96, -80, -96, -90, -96]]


@pytest.mark.parametrize("v_exp", SPREADS)
@pytest.mark.parametrize("queries,dim,page,width,items", [
    (1, 64, 16, None, 1), (1, 128, 64, None, 1), (9, 32, 32, None, 200), (2, 64, 16, None, 300), (60, 64, 16, None, 1),
    (60, 128, 64, None, 1), (200, 32, 128, None, 1), (60, 64, 128, 40, 1)])
def test_pages_at_both_ends_of_the_scales(cuda_device, v_exp, queries, dim, page, width, items):
    """Every token counts in the sum of the weights, however small its page's values are."""
    tokens = 5 * page - 3
    q, k, v = inputs(2, tokens, queries, dim, torch.bfloat16, queries)
    exps = [-7] * 5, v_exp
    got = attend(q, k, v, *exps, page, dim ** -0.5, width=width, items=items)
    check(got, q, k, v, *exps, page, dim ** -0.5)


@pytest.mark.parametrize("queries,dim,page,items", [(1, 64, 16, 1), (1, 64, 16, 900), (3, 128, 64, 700), (60, 64, 16, 1),
                                                    (60, 128, 64, 100)])
@pytest.mark.parametrize("large", [0, 4])
def test_large_values_of_tokens_with_little_weight(cuda_device, queries, dim, page, items, large):
    """The largest page makes the output and the others the sum of the weights: 2^-49 of weight times 2^190."""
    tokens = 5 * page
    q, k, v = inputs(2, tokens, queries, dim, torch.bfloat16, queries)
    scale = dim ** -0.5
    k[:, large * page : (large + 1) * page, 0] = -320
    q.view(queries, 2, dim)[..., 0] = 34 / (5 * scale)
    v_exp = [-96, -95, -96, -94, -96]
    v_exp[large] = 96
    exps = [-6] * 5, v_exp
    got = attend(q, k, v, *exps, page, scale, items=items)
    check(got, q, k, v, *exps, page, scale)
