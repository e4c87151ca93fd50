"""The product's GELU at infinities and in its tails.

Values before the activation are given exactly: rows of zeros, so that only bias and residual count.
The formula's erfc is within 1.5e-7; evaluated in FP32 with the hardware's reciprocal and power of two it
adds 2^-19 of itself.  Half of |y| times that, and one rounding."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, fp8
from oracle import fp8 as oracle
from tests.test_fp8_gpu import TINY, UNIT

pytestmark = pytest.mark.gpu


def zero_rows(m, n, k, dev):
    return fp8.quantize_rows(torch.zeros(m, k, device=dev)), fp8.pack_weight_fp8(torch.ones(n, k, device=dev))


SHAPES = [(40, 64, 256), (1, 40, 8192), (40, 33, 256), (3, 37, 4096), (600, 2304, 2048)]  # one range, ranges, odd rows, CTA pairs


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_infinities_pass_as_the_formula_has_them(cuda_device, dtype, m, n, k):
    """+inf stays, a NaN stays one, and -inf times zero is one: 0.5 y (1 + erf(y / sqrt 2))."""
    rows, weight = zero_rows(m, n, k, cuda_device)
    bias = torch.linspace(-3, 3, n)
    bias[1], bias[2], bias[3], bias[4] = float("inf"), float("-inf"), float("nan"), 3e38
    residual = torch.zeros(m, n, dtype=dtype)
    residual[m - 1, n - 1] = float("inf")
    got = fp8.matmul_fp8(rows, weight, bias.to(cuda_device), residual=residual.to(cuda_device), act=_lib.LDB_ACT_GELU,
                         out_dtype=dtype).cpu()
    zero = torch.zeros(m, k, dtype=torch.float64), torch.zeros(n, k, dtype=torch.float64)
    want = oracle.matmul(*zero, bias, residual, True)[0].to(dtype)
    assert torch.isinf(want[0, 1]) and torch.isnan(want[0, 2]) and torch.isinf(want[m - 1, n - 1])
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_tails(cuda_device, dtype):
    n = 4001
    rows, weight = zero_rows(2, n, 16, cuda_device)
    bias = torch.linspace(-20, 20, n)
    got = fp8.matmul_fp8(rows, weight, bias.to(cuda_device), act=_lib.LDB_ACT_GELU, out_dtype=dtype).cpu().double()
    y = bias.double()
    erfc = torch.special.erfc(y.abs() / 2 ** 0.5)
    want = torch.clamp(y, min=0) - 0.5 * y.abs() * erfc
    bound = (0.5 * y.abs() * (1.5e-7 + 2.0 ** -19 * erfc) + (UNIT[dtype] + 2.0 ** -23) * want.abs() + TINY[dtype])
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
