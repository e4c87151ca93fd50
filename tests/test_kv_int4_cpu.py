"""Paged 4-bit key/value cache: the refusals that need no GPU, and the oracle's own format."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_int4 as oracle


def code(name, args):
    with pytest.raises(_lib.LdbError) as e:
        _lib.call(name, None, *args)
    return e.value.code


def test_library_refuses_bad_caches():
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    append = [p, 64, 64, p, 64, 64, 0, p, p, p, p, 4, 2, 64, 32, p, 4, 4, p, None, 1, 3]
    for at, value, want in ((0, None, -1), (6, 9, -1), (7, None, -1), (18, None, -1), (14, 48, -2), (13, 8, -2),
                            (11, 0, -2), (16, 3, -2), (1, 63, -2), (8, odd, -3), (10, odd, -3), (21, -1, -2),
                            (20, 70000, -2)):
        bad = list(append)
        bad[at] = value
        assert code("ldb_kv_append_int4", bad) == want, (at, value)
    read = [p, p, p, p, 4, 2, 64, 32, p, 4, 4, p, None, p, 64, 192, p, 64, 192, 0, 2, 3]
    for at, value, want in ((0, None, -1), (2, None, -1), (8, None, -1), (11, None, -1), (13, None, -1), (16, None, -1),
                            (19, 5, -1), (7, 16, -2), (6, 8, -2), (4, 0, -2), (9, 3, -2), (14, 63, -2), (15, 63, -2),
                            (18, 0, -2), (0, odd, -3), (20, -1, -2), (20, 70000, -2), (21, -1, -2)):
        bad = list(read)
        bad[at] = value
        for name in ("ldb_kv_read_int4", "ldb_kv_read_fp8"):
            assert code(name, bad) == want, (name, at, value)
    assert code("ldb_kv_read_int4", [*read[:2], odd, *read[3:]]) == -3
    attend = [p, 128, 128, 0, p, p, p, p, 4, 2, 64, 32, p, 4, 4, p, p, 128, 128, 1, 3, 4, 1.0, 0, p, 1 << 40]
    for at, value, want in ((0, None, -1), (3, _lib.LDB_F32, -1), (4, None, -1), (16, None, -1), (21, 5, -2), (11, 96, -2),
                            (10, 24, -2), (8, 0, -2), (13, 3, -2), (1, 127, -2), (17, 127, -2), (5, odd, -3), (6, odd, -3),
                            (19, 2049, -2), (24, None, -4), (25, 16, -4), (24, odd, -4), (8, 1 << 30, -2)):
        bad = list(attend)
        bad[at] = value
        assert code("ldb_kv_attention_int4", bad) == want, (at, value)
    need = ctypes.c_size_t(0)
    with pytest.raises(_lib.LdbError, match="heads"):
        _lib.call("ldb_kv_attention_int4_workspace_size", 1, 1, 3, 2, 64, 100, ctypes.byref(need))


def test_empty_calls_launch_nothing():
    before = _lib.launch_count()
    _lib.call("ldb_kv_append_int4", None, None, 0, 0, None, 0, 0, 0, None, None, None, None, 4, 2, 64, 32, None, 4, 4,
              None, None, 0, 3)
    for batch, tokens in ((0, 3), (2, 0)):
        _lib.call("ldb_kv_read_int4", None, None, None, None, None, 4, 2, 64, 32, None, 4, 4, None, None, None, 0, 0, None,
                  0, 0, 0, batch, tokens)
    _lib.call("ldb_kv_attention_int4", None, None, 0, 0, 0, None, None, None, None, 4, 2, 64, 32, None, 4, 4, None, None,
              0, 0, 0, 3, 4, 1.0, 0, None, 0)
    assert _lib.launch_count() == before


def test_python_refuses_what_does_not_fit():
    with pytest.raises(ValueError, match="pages hold"):
        kv_cache.KvCacheInt4.empty(2, 1, 64, page=65, device="cpu")
    with pytest.raises(ValueError, match="pages hold"):
        kv_cache.KvCacheInt4.empty(2, 1, 80, device="cpu")
    cache = kv_cache.KvCacheInt4.empty(2, 1, 64, device="cpu")
    index = torch.zeros(1, 1, dtype=torch.int32)
    calls = (lambda c: kv_cache.kv_append(c, torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), index, index[0]),
             lambda c: kv_cache.kv_attention(torch.zeros(1, 1, 64), c, index, index[0], scale=1.0),
             lambda c: kv_cache.kv_read(c, index, index[0], tokens=1))
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call(cache)
        with pytest.raises(ValueError, match="uint8"):
            call(cache._replace(v=cache.v.float()))
        with pytest.raises(ValueError, match="scales"):
            call(cache._replace(v_scale=cache.v_scale[:, :, :1]))


def test_format():
    """The oracle's scales are a float16's upper bits, and no value is further than half a scale from its code's."""
    assert len(oracle.SCALES) == 199 and oracle.SCALES[-1] == 896.0
    bits = (torch.arange(199, dtype=torch.int16) << 7).view(torch.float16).double()
    assert torch.equal(bits, torch.tensor(oracle.SCALES, dtype=torch.float64))
    x = torch.randn(400, 16, generator=torch.Generator().manual_seed(1)) * torch.exp2(torch.linspace(-15, 10, 400))[:, None]
    for row in x:
        codes, byte = oracle.quantize(row)
        s = oracle.SCALES[byte]
        assert ((codes.double() - 8) * s - row.double()).abs().max() <= s / 2
        assert 7.5 * oracle.SCALES[byte - 1] < row.double().abs().max() <= 7.5 * s
