"""Paged 8-bit key/value cache: the refusals that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache


def code(name, args):
    with pytest.raises(_lib.LdbError) as e:
        _lib.call(name, None, *args)
    return e.value.code


def test_library_refuses_bad_caches():
    p = ctypes.c_void_p(4096)  # never read: every call below fails before a launch
    odd = ctypes.c_void_p(4104)
    append = [p, 64, 64, p, 64, 64, 0, p, p, p, p, 4, 2, 64, 32, p, 4, 4, p, None, 1, 3]
    for at, value, want in ((0, None, -1), (6, 9, -1), (7, None, -1), (18, None, -1), (14, 48, -2), (13, 8, -2),
                            (11, 0, -2), (16, 3, -2), (1, 63, -2), (8, odd, -3), (21, -1, -2), (20, 40000, -2)):
        bad = list(append)
        bad[at] = value
        assert code("ldb_kv_append_fp8", bad) == want, (at, value)
    attend = [p, 128, 128, 0, p, p, p, p, 4, 2, 64, 32, p, 4, 4, p, p, 128, 128, 1, 3, 4, 1.0, 0, p, 1 << 40]
    for at, value, want in ((0, None, -1), (3, _lib.LDB_F32, -1), (4, None, -1), (16, None, -1), (21, 5, -2), (11, 96, -2),
                            (10, 24, -2), (8, 0, -2), (13, 3, -2), (1, 127, -2), (17, 127, -2), (5, odd, -3),
                            (19, 2049, -2), (24, None, -4), (25, 16, -4), (24, odd, -4), (8, 1 << 30, -2)):
        bad = list(attend)
        bad[at] = value
        assert code("ldb_kv_attention_fp8", bad) == want, (at, value)
    need = ctypes.c_size_t(0)
    with pytest.raises(_lib.LdbError, match="heads"):
        _lib.call("ldb_kv_attention_fp8_workspace_size", 1, 1, 3, 2, 64, ctypes.byref(need))


def test_empty_calls_launch_nothing():
    before = _lib.launch_count()
    _lib.call("ldb_kv_append_fp8", None, None, 0, 0, None, 0, 0, 0, None, None, None, None, 4, 2, 64, 32, None, 4, 4, None,
              None, 0, 3)
    _lib.call("ldb_kv_attention_fp8", None, None, 0, 0, 0, None, None, None, None, 4, 2, 64, 32, None, 4, 4, None, None, 0,
              0, 0, 3, 4, 1.0, 0, None, 0)
    assert _lib.launch_count() == before


def test_python_refuses_what_does_not_fit():
    with pytest.raises(ValueError, match="pages hold"):
        kv_cache.KvCacheFp8.empty(2, 1, 64, page=65, device="cpu")
    with pytest.raises(ValueError, match="pages hold"):
        kv_cache.KvCacheFp8.empty(2, 1, 80, device="cpu")
    cache = kv_cache.KvCacheFp8.empty(2, 1, 64, device="cpu")
    index = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache.kv_append(cache, torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), index, index[0])
    bad = kv_cache.KvCacheFp8(cache.k.float(), cache.v, cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        kv_cache.kv_attention(torch.zeros(1, 1, 64), bad, index, index[0], scale=1.0)
    bad = kv_cache.KvCacheFp8(cache.k, cache.v, cache.k_scale[:1], cache.v_scale)
    with pytest.raises(ValueError, match="scales"):
        kv_cache.kv_attention(torch.zeros(1, 1, 64), bad, index, index[0], scale=1.0)


def test_workspace_of_a_table_is_within_that_of_any():
    def size(name, *args):
        need = ctypes.c_size_t(0)
        _lib.call(name, *args, ctypes.byref(need))
        return need.value

    for batch, queries, heads, kv_heads, dim in ((1, 1, 8, 2, 128), (7, 523, 4, 4, 32), (3, 100, 8, 1, 64), (40, 60, 8, 8, 32),
                                                 (64, 4000, 8, 8, 128)):
        most = size("ldb_kv_attention_fp8_workspace_size", batch, queries, heads, kv_heads, dim)
        for capacity in (16, 77, 1000, 19724, 130000, 2 ** 31 - 1):
            got = size("ldb_kv_attention_fp8_table_workspace_size", batch, queries, heads, kv_heads, dim, capacity)
            assert got <= most, (batch, queries, capacity)
    assert size("ldb_kv_attention_fp8_table_workspace_size", 1, 6400, 4, 4, 64, 77) == 0  # one block: nothing to join
