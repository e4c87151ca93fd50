"""Rows that start at an odd value: written to the 4-bit cache and turned, in every type."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from lesiondiffusion_mlx_b200.rotary import Rotary, qk_norm_rope
from oracle import rotary as oracle
from tests.test_kv_int4_gpu import append_both, host, ints, make_cache, make_table, same_cache
from tests.test_rotary_gpu import check, frequencies

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lo", [0, 1, 2, 3, 8])
def test_written_and_turned(cuda_device, dtype, lo):
    heads, dim, page = 2, 32, 16
    table, pages = make_table(2, 3, 1)
    cache = make_cache(pages, heads, dim, page, cuda_device, 2)
    want = host(cache)
    wide = torch.randn(2, 6, 2 * heads * dim + 9, generator=torch.Generator().manual_seed(lo)).to(dtype)
    k, v = (wide[..., lo + n: lo + n + heads * dim] for n in (0, heads * dim))
    dev = wide.to(cuda_device)
    dev_k, dev_v = (dev[..., lo + n: lo + n + heads * dim] for n in (0, heads * dim))
    kv_cache.kv_append(cache, dev_k, dev_v, table.to(cuda_device), ints([3, 14], cuda_device))
    append_both(want, k, v, table, [3, 14], [6, 6])
    same_cache(cache, want)
    at = torch.arange(12, dtype=torch.int32).view(2, 6)
    for interleaved in (False, True):
        plan = Rotary.build((16,), interleaved=interleaved, device=cuda_device)
        got = qk_norm_rope(dev_k, dev_v, head_dim=dim, rotary=plan, positions=at.to(cuda_device))
        for x, y in zip(got, (k, v)):
            ref = oracle.qk_norm_rope(y, dim, None, 1e-6, True, *frequencies((16,)), interleaved, at[..., None])
            check(x, ref, dim, dtype)
    assert _lib.device_status(reset=True) == 0
