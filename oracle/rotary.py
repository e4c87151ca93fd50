"""Normed and rotated heads in 64 bits, from the definition: each pair a complex number."""

from __future__ import annotations

import torch


def qk_norm_rope(x: torch.Tensor, head_dim: int, gamma: torch.Tensor | None, eps: float, norm: bool,
                 frequencies: list[float], axis: list[int], interleaved: bool, positions: torch.Tensor | None) -> dict:
    """Heads of ``x`` (B, L, n * head_dim), and for an error bound each value's size: its pair's length."""
    y = x.double().unflatten(-1, (-1, head_dim)).clone()
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    if gamma is not None:
        y = y * gamma.double()
    size = y.abs()
    n = len(frequencies)
    for i, (f, a) in enumerate(zip(frequencies, axis)):
        low, high = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        angle = (positions[..., a].double() * f)[..., None]
        z = torch.complex(y[..., low], y[..., high]) * torch.polar(torch.ones_like(angle), angle)
        size[..., low] = size[..., high] = z.abs()
        y[..., low], y[..., high] = z.real, z.imag
    return {"out": y.flatten(-2), "size": size.flatten(-2)}
