"""4-bit cache: numbers that a call's descriptor cannot hold, a scale that is not a number, and the bound on a value's error."""

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
