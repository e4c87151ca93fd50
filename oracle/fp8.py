"""The 8-bit row / weight format, norm and product in 64 bits, from their definitions."""

from __future__ import annotations

import torch

BLOCK = 128
E4M3_MAX = 448.0


def exponent(amax: torch.Tensor) -> torch.Tensor:
    """The least e in [-127, 127] with amax <= 448 * 2^e, 0 for amax = 0 (float64 in, int64 out)."""
    mantissa, power = torch.frexp(amax.double() / 7.0)  # 448 = 7 * 2^6; amax / 7 <= 2^(e + 6)
    e = torch.where(mantissa == 0.5, power - 1, power).to(torch.int64) - 6
    return torch.where(amax == 0, torch.zeros_like(e), e).clamp(-127, 127)


def _amax(y: torch.Tensor, dims) -> torch.Tensor:
    return torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y)).amax(dims)


def to_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, ties to even (|v| <= 448; what is not finite becomes NaN), as float64."""
    a = v.double().abs()
    _, power = torch.frexp(torch.where(torch.isfinite(a), a, torch.ones_like(a)))
    step = torch.exp2((power - 1).clamp(min=-6).double() - 3)
    q = torch.round(v.double() / step) * step  # torch.round: ties to even
    return torch.where(torch.isfinite(v), q, torch.full_like(q, float("nan")))


def quantize_rows(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(code values, exponents) of (rows, k): a scale per row and 128 channels."""
    rows, k = y.shape
    blocks = -(-k // BLOCK)
    padded = torch.nn.functional.pad(y.double(), (0, blocks * BLOCK - k)).view(rows, blocks, BLOCK)
    e = exponent(_amax(padded, -1))
    codes = to_e4m3(padded * torch.exp2(-e.double())[..., None])
    return codes.view(rows, -1)[:, :k], e


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(code values, exponents) of (n, k): a scale per 128 x 128 block."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    padded = torch.nn.functional.pad(w.double(), (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    e = exponent(_amax(padded, (1, 3)))
    codes = to_e4m3(padded * torch.exp2(-e.double())[:, None, :, None])
    return codes.view(nb * BLOCK, kb * BLOCK)[:n, :k], e


def dequantize_rows(codes: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    k = codes.shape[-1]
    return codes.double() * torch.exp2(e.double()).repeat_interleave(BLOCK, -1)[..., :k]


def dequantize_weight(codes: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    n, k = codes.shape
    scale = torch.exp2(e.double()).repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return codes.double() * scale


def rms_norm(x: torch.Tensor, gamma: torch.Tensor | None, residual: torch.Tensor | None, eps: float
             ) -> tuple[torch.Tensor, torch.Tensor]:
    """(h, h * rsqrt(mean(h^2) + eps) * gamma)."""
    h = x.double() + (0 if residual is None else residual.double())
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return h, y if gamma is None else y * gamma.double()


def matmul(a: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None, gelu: bool
           ) -> tuple[torch.Tensor, torch.Tensor]:
    """(act(a w^T + bias + residual), the sum of the terms' magnitudes) of dequantized operands."""
    y, size = a @ w.T, a.abs() @ w.abs().T
    for term in (bias, residual):
        if term is not None:
            y, size = y + term.double(), size + term.double().abs()
    return (0.5 * y * (1 + torch.erf(y / 2 ** 0.5)) if gelu else y), size
