"""Rotary plans, and the refusals of their kernel that need no GPU."""

from __future__ import annotations

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
    p, odd = 4096, 4104
    fields = ("size", "dtype", "q", "k", "q_out", "k_out", "q_ld", "q_batch", "k_ld", "k_batch", "q_out_ld", "q_out_batch",
              "k_out_ld", "k_out_batch", "q_gamma", "k_gamma", "turns", "axis", "positions", "positions_ld",
              "positions_batch", "batch", "tokens", "heads", "kv_heads", "head_dim", "pairs", "axes", "interleaved", "norm",
              "eps")
    desc = _lib.DESCRIPTORS["ldb_qk_norm_rope_desc"]
    good = dict(zip(fields, (desc.size, 0, p, p, p, p, 256, 1024, 128, 512, 256, 1024, 128, 512, p, p, p, p, p, 1, 4, 2, 4,
                             4, 2, 64, 32, 1, 0, 1, 1e-6)))
    for name, value, want in (("q", 0, -1), ("k", 0, -1), ("dtype", 7, -1), ("turns", 0, -1), ("axis", 0, -1),
                              ("positions", 0, -1), ("q_out", 0, -1), ("k_out", 0, -1), ("size", desc.size - 8, -1),
                              ("head_dim", 72, -2), ("head_dim", 272, -2), ("head_dim", 0, -2), ("pairs", 33, -2),
                              ("pairs", 12, -2), ("pairs", -1, -2), ("axes", 0, -2), ("q_ld", 255, -2),
                              ("q_out_ld", 255, -2), ("q_out_batch", 255, -2), ("k_ld", 127, -2), ("batch", -1, -2),
                              ("tokens", -1, -2), ("heads", -4, -2), ("q_gamma", odd, -3), ("k_gamma", odd, -3)):
        with pytest.raises(_lib.LdbError) as e:
            _lib.call("ldb_qk_norm_rope", None, desc.pack(*(good | {name: value}).values()))
        assert e.value.code == want, (name, value)
    with pytest.raises(_lib.LdbError, match="null"):
        _lib.call("ldb_qk_norm_rope", None, None)
    before = _lib.launch_count()
    for name in ("batch", "tokens"):
        _lib.call("ldb_qk_norm_rope", None, desc.pack(*(good | {name: 0}).values()))
    assert _lib.launch_count() == before
