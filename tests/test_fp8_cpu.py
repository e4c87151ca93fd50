"""8-bit format, norm and product: the oracle's own definitions and the refusals that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, fp8
from oracle import fp8 as oracle


def test_oracle_rounds_like_the_type_itself():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    values = codes[torch.isfinite(codes)].sort().values
    mid = (values[1:] + values[:-1]) / 2
    probe = torch.cat([values, mid, mid * (1 + 2 ** -20), mid * (1 - 2 ** -20)]).clamp(-448, 448)
    assert torch.equal(oracle.to_e4m3(probe), probe.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.0 * (1 + 2 ** -20), 1), (224.0, -1), (1.0, -8), (0.0, 0),
                                    (1.75, -8), (1.7500001, -7), (3.0e38, 120), (1.0e-44, -127)])
def test_oracle_exponent_is_the_least_that_fits(amax, e):
    assert int(oracle.exponent(torch.tensor(amax, dtype=torch.float64))) == e
    if 0 < amax and -127 < e:
        assert amax <= 448 * 2.0 ** e and amax > 448 * 2.0 ** (e - 1)


def test_library_refuses_bad_rows_and_products():
    p = ctypes.c_void_p(4096)  # never read: every call below fails before a launch
    odd = ctypes.c_void_p(4097)

    def code(name, *args):
        with pytest.raises(_lib.LdbError) as e:
            _lib.call(name, None, *args)
        return e.value.code

    norm = [p, 64, None, 0, _lib.LDB_F16, None, 1e-6, None, 0, p, 64, p, 4, 2, 64]
    for at, value, want in ((0, None, -1), (4, 7, -1), (14, 0, -2), (14, 32769, -2), (1, 63, -2), (10, 72, -3),
                            (9, odd, -3), (13, -1, -2), (12, 0, -2)):
        bad = list(norm)
        bad[at] = value
        assert code("ldb_rms_norm_fp8", *bad) == want, (at, value)
    assert code("ldb_quantize_fp8_rows", p, 64, 9, p, 64, p, 4, 2, 64) == -1
    assert code("ldb_pack_weight_fp8", p, 64, 0, p, 60, p, 1, 4, 64) == -2
    mm = [p, 128, p, 4, p, 128, p, 1, None, None, 0, p, 32, 8, 32, 128, 0, 0, None, 0]
    for at, value, want in ((0, None, -1), (16, 5, -1), (17, 5, -1), (13, 0, -2), (1, 120, -2), (1, 136, -3),
                            (4, odd, -3), (2, odd, -3), (3, 6, -3), (12, 31, -2), (7, 0, -2)):
        bad = list(mm)
        bad[at] = value
        assert code("ldb_matmul_fp8", *bad) == want, (at, value)
    # few tiles over a long K are split, and the partial sums have to be given a place
    need = ctypes.c_size_t(0)
    _lib.call("ldb_matmul_fp8_workspace_size", 1, 32, 8192, ctypes.byref(need))
    assert need.value > 0
    split = list(mm)
    split[1], split[3], split[5], split[7], split[13], split[15] = 8192, 64, 8192, 64, 1, 8192
    assert code("ldb_matmul_fp8", *split) == -4


def test_python_refuses_what_does_not_fit():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.rms_norm_fp8(x, None)
    with pytest.raises(ValueError, match="float16, bfloat16 or float32"):
        fp8.quantize_rows(torch.zeros(2, 64, dtype=torch.int32))
    rows = fp8.Fp8Rows(x.to(fp8.CODES), torch.ones(2, 1).to(fp8.SCALES))
    weight = fp8.Fp8Weight(x.to(fp8.CODES), torch.ones(1, 1).to(fp8.SCALES))
    with pytest.raises(ValueError, match="CUDA"):
        fp8.matmul_fp8(rows, weight)
    with pytest.raises(ValueError, match="float8"):
        fp8.matmul_fp8(fp8.Fp8Rows(x, rows.scales), weight)


def test_extents_past_32_bits_are_refused_not_wrapped():
    need = ctypes.c_size_t(0)
    for m, n, k in ((2 ** 31 - 1, 8, 128), (8, 2 ** 31 - 1, 128), (8, 8, 2 ** 31 - 1)):
        with pytest.raises(_lib.LdbError) as e:
            _lib.call("ldb_matmul_fp8_workspace_size", m, n, k, ctypes.byref(need))
        assert e.value.code == -2
    with pytest.raises(ValueError, match="at most"):
        fp8._flat(torch.zeros(1, 1).expand(2 ** 32 + 1, 1), "x")
    with pytest.raises(ValueError, match="at most"):
        fp8._flat(torch.zeros(1, 1, 1).expand(2 ** 16, 2 ** 16, 1), "x")
