"""Paged 4-bit key/value cache: the refusals that need no GPU, and the oracle's own format."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, kv_cache
from oracle import kv_int4 as oracle


P, ODD = 4096, 4104
CACHE = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, table=P, table_ld=4, pages=4, kv_heads=2, page=64, head_dim=32,
             width=4, batch=1)


def descriptors():
    """A good call of each operator, by field in the descriptor's order."""
    size = {n: _lib.DESCRIPTORS[f"ldb_kv_{n}_desc"].size for n in ("append", "read", "attention")}
    rows = dict(k_ld=64, k_batch=192, v_ld=64, v_batch=192)
    return {"append": dict(size=size["append"], dtype=0) | CACHE | dict(k=P, v=P) | rows | dict(start=P, counts=0, tokens=3),
            "read": dict(size=size["read"], dtype=0) | CACHE | dict(k=P, v=P) | rows | dict(lengths=P, start=0, tokens=3),
            "attention": dict(size=size["attention"], dtype=0) | CACHE | dict(
                q=P, out=P, q_ld=128, q_batch=384, out_ld=128, out_batch=384, lengths=P, workspace=P,
                workspace_bytes=1 << 40, queries=3, heads=4, causal=0, scale=1.0)}


def call(name, fields, bits="int4"):
    _lib.call(f"ldb_kv_{name}_{bits}", None, _lib.DESCRIPTORS[f"ldb_kv_{name}_desc"].pack(*fields.values()))


SHARED = (("k_codes", 0, -1), ("v_scales", 0, -1), ("table", 0, -1), ("page", 48, -2), ("page", 8, -2), ("head_dim", 24, -2),
          ("pages", 0, -2), ("table_ld", 3, -2), ("width", 0, -2), ("k_codes", ODD, -3), ("batch", -1, -2), ("dtype", 9, -1),
          ("size", 8, -1))


@pytest.mark.parametrize("name,bits,cases", [
    ("append", "int4", (("k", 0, -1), ("start", 0, -1), ("k_ld", 63, -2), ("k_scales", ODD, -3), ("tokens", -1, -2),
                        ("batch", 70000, -2))),
    ("read", "int4", (("v", 0, -1), ("lengths", 0, -1), ("k_ld", 63, -2), ("v_ld", 63, -2), ("tokens", -1, -2),
                      ("batch", 70000, -2), ("v_scales", ODD, -3))),
    ("read", "fp8", (("v", 0, -1), ("lengths", 0, -1), ("k_ld", 63, -2), ("tokens", -1, -2))),
    ("attention", "int4", (("q", 0, -1), ("dtype", _lib.LDB_F32, -1), ("lengths", 0, -1), ("out", 0, -1), ("heads", 5, -2),
                           ("q_ld", 127, -2), ("out_ld", 127, -2), ("v_scales", ODD, -3), ("batch", 2049, -2),
                           ("workspace", 0, -4), ("workspace_bytes", 16, -4), ("workspace", ODD, -4), ("pages", 1 << 30, -2), ("pages", (1 << 31) - 1, -2),
                           ("queries", -1, -2), ("kv_heads", 0, -2)))])
def test_library_refuses_bad_calls(name, bits, cases):
    good = descriptors()[name]
    for field, value, want in SHARED + cases:
        with pytest.raises(_lib.LdbError) as e:
            call(name, good | {field: value}, bits)
        assert e.value.code == want, (field, value)
    with pytest.raises(_lib.LdbError, match="null"):
        _lib.call(f"ldb_kv_{name}_{bits}", None, None)


def test_item_strides_of_what_is_written():
    good = descriptors()
    for name, field in (("read", "v_batch"), ("attention", "out_batch")):
        with pytest.raises(_lib.LdbError, match="item stride"):
            call(name, good[name] | {"batch": 2, field: 0})
    need = ctypes.c_size_t(0)
    with pytest.raises(_lib.LdbError, match="heads"):
        _lib.call("ldb_kv_attention_int4_workspace_size", 1, 1, 3, 2, 64, 100, ctypes.byref(need))


def test_tables_past_the_last_block():
    # 2^31 - 256 tokens: the number of the token behind a last block of 128 still has a sign to spare
    attention = descriptors()["attention"] | dict(page=16, width=0x7FFFFF1, table_ld=0x7FFFFF1)
    with pytest.raises(_lib.LdbError, match="table of") as e:
        call("attention", attention)
    assert e.value.code == -2


def test_numbers_past_their_fields():
    desc = _lib.DESCRIPTORS["ldb_kv_attention_desc"]
    fields = list(descriptors()["attention"].values())[1:]
    assert _lib.packed("kv_attention", desc, *fields) == desc.pack(desc.size, *fields)
    for at, value in ((-4, 2 ** 31), (-4, 1.5), (-1, None)):
        with pytest.raises(ValueError, match="kv_attention"):
            _lib.packed("kv_attention", desc, *fields[:at], value, *(fields[at + 1:] if at + 1 else []))


def test_empty_calls_launch_nothing():
    before, good = _lib.launch_count(), descriptors()
    for name, field in (("append", "batch"), ("append", "tokens"), ("read", "batch"), ("read", "tokens"),
                        ("attention", "batch"), ("attention", "queries")):
        call(name, good[name] | {field: 0})
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
