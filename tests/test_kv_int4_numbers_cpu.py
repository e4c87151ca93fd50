"""4-bit cache: scales that are not finite numbers, and the bound on the error of a value."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib
from oracle import kv_int4 as oracle
from tests.test_kv_int4_cpu import call, descriptors


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3.0e38])
def test_attention_refuses_scales_that_are_not_finite(scale):
    """(3e38 is past FP32 as a power of two's factor.)"""
    with pytest.raises(_lib.LdbError, match="scale") as e:
        call("attention", descriptors()["attention"] | {"scale": scale})
    assert e.value.code == -1


def test_error_of_a_value():
    """Half the scale that is taken: a 15th of the group's largest and an eighth more while scales have a leading bit, and
    2^-18 more below (the statement of ``kv_append``)."""
    g = torch.Generator().manual_seed(1)
    past_an_eighth = 0
    for top in torch.exp2(torch.linspace(-20, -9, 1200, dtype=torch.float64)).tolist():
        x = top * (2 * torch.rand(16, generator=g, dtype=torch.float64) - 1)
        x[3] = top
        codes, byte = oracle.quantize(x)
        error = float(((codes.double() - 8) * oracle.SCALES[byte] - x).abs().max())
        assert error <= max(top / 15 * 9 / 8, top / 15 + 2.0 ** -18)
        past_an_eighth += error > top / 15 * 9 / 8
    assert past_an_eighth
