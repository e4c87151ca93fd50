"""What decides a page's scale where the new values say little or too much."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_cache as oracle
from tests.test_kv_cache_gpu import host, ints, make_cache, make_table, same_cache

pytestmark = pytest.mark.gpu

LAYOUTS = [(2, 32, 16), (1, 64, 64), (3, 128, 64), (1, 128, 128)]  # heads, channels, page


@pytest.mark.parametrize("heads,dim,page", LAYOUTS)
@pytest.mark.parametrize("value", [0.0, float("nan"), float("inf")])
def test_tokens_without_a_finite_value_leave_the_older_ones_alone(cuda_device, heads, dim, page, value):
    """A token of zeros, NaN or infinities behind older ones keeps the page's scale and its codes; in a page
    of its own it has the scale 1."""
    table, pages = make_table(2, 2, cuda_device, 3)
    cache = make_cache(pages, heads, dim, page, cuda_device, 4, low=-20, high=-5)
    want = host(cache)
    start = [page - 3, page]
    new = torch.full((2, 2, heads * dim), value, dtype=torch.bfloat16)
    kv_cache.kv_append(cache, new.to(cuda_device), new.to(cuda_device), table.to(cuda_device), ints(start, cuda_device))
    first, own = int(table[0, 0]), int(table[1, 1])
    for codes, e in ((want[0], want[1]), (want[2], want[3])):
        codes[first, :, page - 3 : page - 1] = codes[own, :, :2] = 0 if value == 0 else float("nan")
        e[own] = 0
    same_cache(cache, want)
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("heads,dim,page", LAYOUTS)
def test_scales_stay_within_their_bounds(cuda_device, heads, dim, page):
    """Past 448 * 2^96 a value saturates; under 2^-96 * 2^-10 it is zero."""
    table, pages = make_table(1, 3, cuda_device, 5)
    cache = make_cache(pages, heads, dim, page, cuda_device, 6)
    new = torch.ones(1, 2 * page, heads * dim)
    new[0, :page] = 1e35
    new[0, 0], new[0, 1] = -3e38, 448 * 2.0 ** 96 / 2
    new[0, page:] = 2.0 ** -104
    new[0, page + 1] = 2.0 ** -107
    kv_cache.kv_append(cache, new.to(cuda_device), new.to(cuda_device), table.to(cuda_device), ints([0], cuda_device))
    for codes, e in (host(cache)[:2], host(cache)[2:]):
        large, small = int(table[0, 0]), int(table[0, 1])
        assert (e[large] == 96).all() and (e[small] == -96).all()
        assert (codes[large, :, 0] == -448).all() and (codes[large, :, 1] == 224).all() and (codes[large, :, 2:] == 448).all()
        assert (codes[small, :, 0] == 2.0 ** -8).all() and (codes[small, :, 1] == 0).all()
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("dim,page", [(128, 32), (64, 64), (32, 128), (128, 64), (64, 128), (128, 128)])
@pytest.mark.parametrize("fewer", [0, 1])
def test_calls_of_a_page_and_of_one_token_less(cuda_device, dtype, dim, page, fewer):
    """Both sides of the number of tokens that decides how a page is shared out."""
    heads, tokens, start = 2, page - fewer, [0, 5]
    table, pages = make_table(2, 3, cuda_device, 7)
    cache = make_cache(pages, heads, dim, page, cuda_device, 8)
    want = host(cache)
    g = torch.Generator().manual_seed(page + dim)
    k, v = ((torch.randn(2, tokens, heads * dim, generator=g) * 30).to(dtype) for _ in range(2))
    kv_cache.kv_append(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), ints(start, cuda_device))
    for (codes, e), new in zip(((want[0], want[1]), (want[2], want[3])), (k, v)):
        oracle.append(codes, e, new.view(2, tokens, heads, dim), table, start, [tokens] * 2)
    same_cache(cache, want)
    assert _lib.device_status(reset=True) == 0
