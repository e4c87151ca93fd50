"""Positions for token blocks: each head's queries and keys normed and rotated in one pass.

Pairs of a head's channels turn by angles that grow with the token's position,
along one axis (a sequence) or several (a volume's depth, height and width, each
with its own share of the channels):

    plan = Rotary.build((16, 24, 24), device="cuda")           # 64 channels: depth, height, width
    at = grid_positions(16, 20, 20, device="cuda")             # of a (B, 6400, C) volume's tokens
    q, k = qk_norm_rope(q, k, head_dim=64, q_gamma=qg, k_gamma=kg, rotary=plan, positions=at)

A plan holds a position's share of a full turn as a 64-bit fraction, rounded once, whose product
with a position is exact: an angle is within 2^-25 of a turn at any 32-bit position.  Inputs are channels-last ``torch`` CUDA tensors;
the call checks shapes, dtypes and devices and launches on the current stream.
"""

from __future__ import annotations

import decimal
import functools
import math
from fractions import Fraction
from typing import NamedTuple, Sequence

import torch

from . import _lib
from .fp8 import _check_input, _launcher, _raw_stream
from .ops import _DT

_current_device = torch._C._cuda_getDevice


@functools.lru_cache
def _full_turn(bits: int) -> int:
    """2 pi * 2^bits, within one (Machin: pi / 4 = 4 atan(1/5) - atan(1/239))."""
    one = 1 << (bits + 32)

    def atan_of_inverse(n: int) -> int:
        total, term, k = 0, one // n, 0
        while term:
            total += (term // (2 * k + 1)) * (-1) ** k
            term, k = term // (n * n), k + 1
        return total

    return 8 * (4 * atan_of_inverse(5) - atan_of_inverse(239)) >> 32


def _turns(frequency: Fraction) -> int:
    """``frequency / (2 pi)`` modulo 1 as a 64-bit fraction, rounded to nearest.

    (In doubles it has 53 bits: 100 radians a step are off by 2^-21 of a turn at position 2^31.)"""
    bits = 160 + max(0, abs(frequency.numerator).bit_length() - frequency.denominator.bit_length())
    n, d = frequency.numerator << (64 + bits), frequency.denominator * _full_turn(bits)
    return (2 * n + d) // (2 * d) % 2 ** 64


class Rotary(NamedTuple):
    """Which pairs of a head's channels turn, how fast, and along which axis.

    Pair ``i`` of ``len(turns)`` is channels ``(i, i + len(turns))``, or ``(2i, 2i + 1)``
    with ``interleaved``; it turns by ``turns[i] / 2^64`` (int64, as the unsigned
    number of the same bits) of a full turn for each step along axis ``axis[i]`` (int32).
    Channels behind the pairs stay as they are."""

    turns: torch.Tensor
    axis: torch.Tensor
    axes: int = 1
    interleaved: bool = False

    @classmethod
    def from_frequencies(cls, frequencies: Sequence[float | Fraction], axis: Sequence[int] | None = None, *,
                         interleaved: bool = False, device: torch.device | str = "cuda") -> "Rotary":
        """Pairs of these frequencies (radians a step), all along one axis where ``axis`` is not given."""
        axis = [0] * len(frequencies) if axis is None else [int(a) for a in axis]
        if len(axis) != len(frequencies) or not axis or min(axis) < 0:
            raise ValueError(f"Rotary: {len(frequencies)} frequencies along {len(axis)} axes")
        exact = [f if isinstance(f, Fraction) else float(f) for f in frequencies]
        if not all(isinstance(f, Fraction) or math.isfinite(f) for f in exact):
            raise ValueError("Rotary: frequencies must be finite")
        turns = [_turns(Fraction(f)) for f in exact]
        return cls(torch.tensor([t - 2 ** 64 * (t >> 63) for t in turns], dtype=torch.int64, device=device),
                   torch.tensor(axis, dtype=torch.int32, device=device), max(axis) + 1, interleaved)

    @classmethod
    def build(cls, dims: Sequence[int], *, base: float = 10000.0, interleaved: bool = False,
              device: torch.device | str = "cuda") -> "Rotary":
        """``dims[a]`` channels (an even number) along axis ``a``, pair ``i`` of an axis at ``base^(-2 i / dims[a])``."""
        if not dims or any(d < 0 or d % 2 for d in dims) or not base > 0:
            raise ValueError(f"Rotary: {tuple(dims)} channels along the axes (even numbers), base {base}")
        with decimal.localcontext() as context:
            context.prec = 50
            pairs = [(Fraction(decimal.Decimal(base) ** (decimal.Decimal(-2 * i) / d)), a)
                     for a, d in enumerate(dims) for i in range(d // 2)]
        plan = cls.from_frequencies([f for f, _ in pairs], [a for _, a in pairs], interleaved=interleaved, device=device)
        return plan._replace(axes=len(dims))


def grid_positions(*sizes: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """``(1, tokens, axes)`` int32 positions of a volume's voxels in memory order."""
    lines = [torch.arange(n, dtype=torch.int32, device=device) for n in sizes]
    return torch.stack(torch.meshgrid(*lines, indexing="ij"), -1).reshape(1, -1, len(sizes))


_DESC = _lib.DESCRIPTORS["ldb_qk_norm_rope_desc"]


def _check_rows(t: torch.Tensor, like: torch.Tensor, index: int, head_dim: int, name: str) -> tuple[int, ...]:
    """(channels, row stride, item stride, tokens, items)."""
    if t.ndim == 3 and t.dtype is like.dtype and t.get_device() == index:
        (items, tokens, channels), (batch, ld, step) = t.shape, t.stride()
        if channels % head_dim or (step != 1 and channels > 1):
            raise ValueError(f"qk_norm_rope: {name} must hold heads of {head_dim} channels with unit stride")
        return channels, ld, batch, tokens, items
    raise ValueError(f"qk_norm_rope: {name} must be (B, L, n * {head_dim}) of q's dtype, device, B and L")


def _check_gamma(gamma: torch.Tensor | None, like: torch.Tensor, head_dim: int, name: str) -> int:
    if gamma is None:
        return 0
    if (gamma.dtype != torch.float32 or gamma.shape != (head_dim,) or not gamma.is_contiguous()
            or gamma.get_device() != like.get_device()):
        raise ValueError(f"qk_norm_rope: {name} must be contiguous float32 ({head_dim},) on q's device")
    return gamma.data_ptr()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, *, head_dim: int, q_gamma: torch.Tensor | None = None,
                 k_gamma: torch.Tensor | None = None, eps: float = 1e-6, norm: bool = True,
                 rotary: Rotary | None = None, positions: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Queries and keys ``(B, L, n * head_dim)``, head by head normed and rotated, rounded once.

    A head becomes ``x * rsqrt(mean(x^2) + eps) * gamma`` (without ``norm``
    ``x * gamma``; a missing gamma is ones), then its pairs turn by the token's
    ``positions``: int32 ``(B, L, axes)``, ``(1, L, axes)`` for all items, or without the
    last axis where there is one.  Channels are a multiple of 16 up to 256 a
    head; pairs that are not interleaved come in eights.  float16, bfloat16 or float32, any row
    and item stride; ``k`` may be None, and ``q_out`` / ``k_out`` may be ``q`` / ``k``."""
    _check_input(q, "qk_norm_rope: q")
    index = q.get_device()
    if index != _current_device():
        with torch.cuda.device(index):
            return qk_norm_rope(q, k, head_dim=head_dim, q_gamma=q_gamma, k_gamma=k_gamma, eps=eps, norm=norm,
                                rotary=rotary, positions=positions, q_out=q_out, k_out=k_out)
    if head_dim < 16 or head_dim > 256 or head_dim % 16:
        raise ValueError(f"qk_norm_rope: heads have a multiple of 16 channels up to 256, got {head_dim}")
    channels, q_ld, q_batch, tokens, batch = _check_rows(q, q, index, head_dim, "q")
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        qo_ld, qo_batch = channels, tokens * channels
    else:
        if q_out.shape != q.shape:
            raise ValueError("qk_norm_rope: q_out must have q's shape")
        _, qo_ld, qo_batch, _, _ = _check_rows(q_out, q, index, head_dim, "q_out")
    k_ptr = ko_ptr = k_channels = k_ld = k_batch = ko_ld = ko_batch = 0
    if k is not None:
        k_channels, k_ld, k_batch, k_tokens, k_items = _check_rows(k, q, index, head_dim, "k")
        if k_tokens != tokens or k_items != batch:
            raise ValueError(f"qk_norm_rope: k must be (B, L, n * {head_dim}) of q's dtype, device, B and L")
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
            ko_ld, ko_batch = k_channels, tokens * k_channels
        else:
            if k_out.shape != k.shape:
                raise ValueError("qk_norm_rope: k_out must have k's shape")
            _, ko_ld, ko_batch, _, _ = _check_rows(k_out, q, index, head_dim, "k_out")
        k_ptr, ko_ptr = k.data_ptr(), k_out.data_ptr()
    elif k_out is not None:
        raise ValueError("qk_norm_rope: k_out without k")
    turns_ptr = axis_ptr = at_ptr = pairs = axes = at_ld = at_batch = interleaved = 0
    if rotary is not None:
        turns, axis, axes, interleaved = rotary
        pairs = turns.numel()
        if (turns.dtype is not torch.int64 or axis.dtype is not torch.int32 or turns.ndim != 1 or axis.ndim != 1
                or axis.numel() != pairs or not turns.is_contiguous() or not axis.is_contiguous()
                or turns.get_device() != index or axis.get_device() != index):
            raise ValueError("qk_norm_rope: a plan is int64 turns and int32 axes of its pairs, on q's device")
        if 2 * pairs > head_dim or (not interleaved and pairs % 8):
            raise ValueError(f"qk_norm_rope: {pairs} pairs in heads of {head_dim} channels (in eights, where not interleaved)")
        if positions is None or positions.dtype != torch.int32 or positions.get_device() != index:
            raise ValueError("qk_norm_rope: positions must be int32 on q's device")
        at, step = positions.shape, positions.stride()
        if len(at) == 2 and axes == 1:
            at, step = (*at, 1), (*step, 1)
        if (len(at) != 3 or at[0] not in (1, batch) or at[1] != tokens or at[2] != axes
                or (axes > 1 and step[2] != 1)):
            raise ValueError(f"qk_norm_rope: positions must be ({batch} or 1, {tokens}, {axes}), got "
                             f"{tuple(positions.shape)}")
        at_ld, at_batch = step[1], step[0] if at[0] > 1 else 0
        turns_ptr, axis_ptr, at_ptr = turns.data_ptr(), axis.data_ptr(), positions.data_ptr()
    elif positions is not None:
        raise ValueError("qk_norm_rope: positions without a plan")
    _launcher("qk_norm_rope")("ldb_qk_norm_rope", _raw_stream(index), _lib.packed(
        "qk_norm_rope", _DESC, _DT[q.dtype], q.data_ptr(), k_ptr, q_out.data_ptr(), ko_ptr, q_ld, q_batch, k_ld, k_batch, qo_ld,
        qo_batch, ko_ld, ko_batch, _check_gamma(q_gamma, q, head_dim, "q_gamma"),
        _check_gamma(k_gamma, q, head_dim, "k_gamma"), turns_ptr, axis_ptr, at_ptr, at_ld, at_batch, batch, tokens,
        channels // head_dim, k_channels // head_dim, head_dim, pairs, axes, int(interleaved), int(norm), eps))
    return q_out, k_out
