"""Rotary plans, and the refusals of their kernel that need no GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib
from lesiondiffusion_mlx_b200.rotary import Rotary, grid_positions, qk_norm_rope


def test_plans_hold_turns():
    plan = Rotary.build((4, 0, 2), base=100.0, interleaved=True, device="cpu")
    assert plan.axes == 3 and plan.interleaved and plan.axis.tolist() == [0, 0, 2]
    for t, f in zip(plan.turns.tolist(), (1.0, 0.1, 1.0)):
        assert abs(t % 2 ** 64 / 2 ** 64 - f / (2 * math.pi)) < 2.0 ** -53
    back, fast = Rotary.from_frequencies([-0.5, 100.0], device="cpu").turns.tolist()
    assert abs(back / 2 ** 64 + 0.5 / (2 * math.pi)) < 2.0 ** -53
    assert abs(fast % 2 ** 64 / 2 ** 64 - 100 / (2 * math.pi) % 1) < 2.0 ** -48


def test_plans_refuse_what_does_not_fit():
    for make in (lambda: Rotary.build((3,), device="cpu"), lambda: Rotary.build((), device="cpu"),
                 lambda: Rotary.build((4,), base=0.0, device="cpu"), lambda: Rotary.from_frequencies([], device="cpu"),
                 lambda: Rotary.from_frequencies([1.0], [0, 1], device="cpu"),
                 lambda: Rotary.from_frequencies([1.0], [-1], device="cpu"),
                 lambda: Rotary.from_frequencies([float("nan")], device="cpu")):
        with pytest.raises(ValueError, match="Rotary"):
            make()
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(torch.zeros(1, 1, 32), None, head_dim=32)


def test_grid_positions_count_in_memory_order():
    at = grid_positions(2, 3, device="cpu")
    assert at.dtype == torch.int32 and at.tolist() == [[[0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]]


def test_library_refuses_bad_calls():
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    good = [p, 256, 1024, p, 128, 512, 0, p, p, 1e-6, 1, p, p, 32, 1, 0, p, 1, 4, p, 256, 1024, p, 128, 512, 2, 4, 4, 2, 64]
    for at, value, want in ((0, None, -1), (3, None, -1), (6, 7, -1), (11, None, -1), (12, None, -1), (16, None, -1),
                            (19, None, -1), (22, None, -1), (29, 72, -2), (29, 272, -2), (29, 0, -2), (13, 33, -2),
                            (13, 12, -2), (13, -1, -2), (14, 0, -2), (1, 255, -2), (20, 255, -2), (21, 255, -2),
                            (4, 127, -2), (25, -1, -2), (26, -1, -2), (27, -4, -2), (7, odd, -3), (8, odd, -3)):
        bad = list(good)
        bad[at] = value
        with pytest.raises(_lib.LdbError) as e:
            _lib.call("ldb_qk_norm_rope", None, *bad)
        assert e.value.code == want, (at, value)
    before = _lib.launch_count()
    for at in (25, 26):
        empty = list(good)
        empty[at] = 0
        _lib.call("ldb_qk_norm_rope", None, *empty)
    assert _lib.launch_count() == before
