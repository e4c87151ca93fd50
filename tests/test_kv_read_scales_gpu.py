"""Reading an 8-bit cache back under every page scale: exact in 64 bits, rounded once, byte 255 a NaN."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_every_page_scale(cuda_device, dtype):
    pages, page, dim = 256, 16, 32
    codes = torch.arange(page * dim, dtype=torch.int32).remainder(256).to(torch.uint8).view(1, 1, page, dim).repeat(pages, 1, 1, 1)
    scales = torch.arange(pages, dtype=torch.uint8).view(pages, 1)
    k, k_scale = codes.to(cuda_device).view(kv_cache.CODES), scales.to(cuda_device).view(kv_cache.SCALES)
    cache = kv_cache.KvCacheFp8(k, k.clone(), k_scale, k_scale.flip(0).contiguous())
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    lengths = torch.tensor([pages * page], dtype=torch.int32, device=cuda_device)
    got = kv_cache.kv_read(cache, table, lengths, tokens=pages * page, dtype=dtype)
    powers = torch.exp2(scales.double() - 127)
    powers[255] = float("nan")
    for x, s in zip(got, (powers, powers.flip(0))):
        want = (codes.view(torch.float8_e4m3fn).double() * s[..., None, None]).view(1, -1, dim).to(dtype)
        assert torch.equal(torch.isnan(x.cpu()), torch.isnan(want))
        assert torch.equal(x.cpu().nan_to_num(0.0), want.nan_to_num(0.0))
    assert _lib.device_status(reset=True) == 0
