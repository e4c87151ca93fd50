"""Rotary plans against exact rationals at far positions.

A fraction rounded to nearest is off by 2^-65 of a turn, so position p is off by p 2^-65: 2^-34 at 2^31."""

from __future__ import annotations

import decimal
from fractions import Fraction

import pytest

from lesiondiffusion_mlx_b200.rotary import Rotary

PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798214808651")
POSITIONS = (1, 131071, 2 ** 31 - 1, -(2 ** 31))


def off(turns: int, frequency: Fraction, position: int) -> Fraction:
    """How far the plan's angle is from frequency * position, in turns."""
    distance = (Fraction(turns * position, 2 ** 64) - frequency * position / (2 * PI)) % 1
    return min(distance, 1 - distance)


@pytest.mark.parametrize("frequency", [1.0, 100.0, -0.5, 0.1, 1e-9, 12345.678, 2.0 ** -40, -3.0e9, 1e40])
def test_frequencies_keep_64_bits(frequency):
    (turns,) = Rotary.from_frequencies([frequency], device="cpu").turns.tolist()
    for p in POSITIONS:
        assert off(turns, Fraction(frequency), p) <= abs(p) * Fraction(1, 2 ** 65), p


@pytest.mark.parametrize("dims,base", [((128,), 10000.0), ((64,), 500000.0), ((16, 24, 24), 10000.0), ((6,), 0.5)])
def test_built_plans_keep_64_bits(dims, base):
    plan = Rotary.build(dims, base=base, device="cpu").turns.tolist()
    with decimal.localcontext() as context:
        context.prec = 80
        logarithm = decimal.Decimal(base).ln()
        exact = [Fraction((logarithm * -2 * i / d).exp()) for d in dims for i in range(d // 2)]
    assert len(plan) == len(exact)
    for turns, f in zip(plan, exact):
        for p in POSITIONS:
            assert off(turns, f, p) <= abs(p) * (Fraction(1, 2 ** 65) + Fraction(1, 2 ** 120)), (f, p)


def test_frequencies_of_other_kinds():
    want = Rotary.from_frequencies([3.0, 0.5], device="cpu").turns.tolist()
    assert Rotary.from_frequencies([3, Fraction(1, 2)], device="cpu").turns.tolist() == want
    assert Rotary.build((4,), base=float("inf"), device="cpu").turns.tolist() == Rotary.from_frequencies(
        [1.0, 0.0], device="cpu").turns.tolist()
    for base in (float("nan"), -1.0, 0.0):
        with pytest.raises(ValueError, match="base"):
            Rotary.build((4,), base=base, device="cpu")
