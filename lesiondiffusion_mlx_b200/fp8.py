"""8-bit dense path: root-mean-square norm, row quantization and block-scaled products.

Values are e4m3 codes with one power-of-two scale (E8M0) per block: the
smallest ``2^e`` with ``max|y| <= 448 * 2^e`` over the block's finite values.
Rows carry a scale per 128 channels, weights a scale per 128 x 128 block, so
the tensor core applies both inside the product.  A block over tokens reads

    rows, h = rms_norm_fp8(x, gamma, residual=h)      # norm, residual and codes in one pass
    y = matmul_fp8(rows, weight, bias, act=LDB_ACT_GELU)

with ``weight = pack_weight_fp8(w)`` made once.  Inputs are channels-last
``torch`` CUDA tensors; each function checks shapes, dtypes and alignment and
launches on the current stream.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib, instrument
from .ops import _DT, _ptr, _rows, _stream

BLOCK = 128  # channels per scale of a row; rows and channels per scale of a weight
CODES = torch.float8_e4m3fn
SCALES = torch.float8_e8m0fnu


@dataclass(frozen=True)
class Fp8Rows:
    """``(..., K)`` e4m3 codes and ``(..., ceil(K / 128))`` E8M0 scales.

    Code rows are 16-byte aligned (row stride a multiple of 16), scale rows
    4-byte aligned (row stride a multiple of 4)."""

    codes: torch.Tensor
    scales: torch.Tensor


@dataclass(frozen=True)
class Fp8Weight:
    """``(N, K)`` e4m3 codes (row stride a multiple of 16) and ``(ceil(N / 128), ceil(K / 128))`` E8M0 scales."""

    codes: torch.Tensor
    scales: torch.Tensor


def _blocks(k: int) -> int:
    return -(-k // BLOCK)


def _empty_rows(lead: tuple[int, ...], k: int, device: torch.device) -> Fp8Rows:
    codes = torch.empty((*lead, -(-k // 16) * 16), dtype=CODES, device=device)
    blocks = _blocks(k)
    scales = torch.empty((*lead, -(-blocks // 4) * 4), dtype=SCALES, device=device)
    return Fp8Rows(codes if codes.shape[-1] == k else codes[..., :k],
                   scales if scales.shape[-1] == blocks else scales[..., :blocks])


def _flat(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, channels, row stride) of a channels-last tensor dense over its rows."""
    if t.ndim == 2:
        if t.stride(1) != 1 and t.shape[1] != 1:
            raise ValueError(f"{name}: channel axis must have unit stride")
        rows, k = t.shape
        return rows, k, max(t.stride(0), k) if rows <= 1 else t.stride(0)
    if t.ndim < 2:
        raise ValueError(f"{name}: expected (..., channels) with at least two axes")
    per, k, ld = _rows(t)
    rows = t.shape[0] * per
    if t.shape[0] > 1 and per and t.stride(0) != per * ld:
        raise ValueError(f"{name}: tensor must be dense over its rows")
    return rows, k, max(ld, k) if rows <= 1 else ld


def _check_input(x: torch.Tensor, name: str) -> None:
    if x.dtype not in _DT:
        raise ValueError(f"{name} must be float16, bfloat16 or float32, got {x.dtype}")
    if x.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor")


def rms_norm_fp8(x: torch.Tensor, gamma: torch.Tensor | None, *, residual: torch.Tensor | None = None,
                 eps: float = 1e-6) -> tuple[Fp8Rows, torch.Tensor]:
    """``h = x + residual`` and the 8-bit rows of ``h * rsqrt(mean(h^2) + eps) * gamma``.

    The sum, the norm and the maximum of a block are FP32, of the unrounded
    ``h``; the returned ``h`` is rounded to ``x``'s dtype (without a residual it
    is ``x`` itself).  ``x`` is ``(..., C)`` float16 / bfloat16 / float32 of up
    to 32768 channels, ``gamma`` float32 ``(C,)``."""
    _check_input(x, "rms_norm_fp8: x")
    rows, c, x_ld = _flat(x, "rms_norm_fp8: x")
    if gamma is not None and (gamma.dtype != torch.float32 or gamma.shape != (c,) or not gamma.is_contiguous()
                              or gamma.device != x.device):
        raise ValueError(f"rms_norm_fp8: gamma must be contiguous float32 ({c},) on x's device")
    h, h_ld, r_ld = None, 0, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError("rms_norm_fp8: residual must have x's shape, dtype and device")
        _, _, r_ld = _flat(residual, "rms_norm_fp8: residual")
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        h_ld = c
    out = _empty_rows(tuple(x.shape[:-1]), c, x.device)
    with instrument.maybe_time("rms_norm_fp8", 0.0):
        _lib.call("ldb_rms_norm_fp8", _stream(x), x.data_ptr(), x_ld, _ptr(residual), r_ld, _DT[x.dtype], _ptr(gamma),
                  eps, _ptr(h), h_ld, out.codes.data_ptr(), -(-c // 16) * 16, out.scales.data_ptr(),
                  -(-_blocks(c) // 4) * 4, rows, c)
    return out, x if h is None else h


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """8-bit rows of ``(..., K)`` float16 / bfloat16 / float32 ``x`` (up to 32768 channels)."""
    _check_input(x, "quantize_rows: x")
    rows, k, x_ld = _flat(x, "quantize_rows: x")
    out = _empty_rows(tuple(x.shape[:-1]), k, x.device)
    with instrument.maybe_time("quantize_rows", 0.0):
        _lib.call("ldb_quantize_fp8_rows", _stream(x), x.data_ptr(), x_ld, _DT[x.dtype], out.codes.data_ptr(),
                  -(-k // 16) * 16, out.scales.data_ptr(), -(-_blocks(k) // 4) * 4, rows, k)
    return out


def pack_weight_fp8(weight: torch.Tensor) -> Fp8Weight:
    """8-bit form of an ``(N, K)`` float16 / bfloat16 / float32 dense weight (once per weight)."""
    _check_input(weight, "pack_weight_fp8: weight")
    if weight.ndim != 2 or 0 in weight.shape:
        raise ValueError(f"pack_weight_fp8: expected an (N, K) weight, got {tuple(weight.shape)}")
    n, k, ld = _flat(weight, "pack_weight_fp8: weight")
    codes = torch.zeros((n, -(-k // 16) * 16), dtype=torch.uint8, device=weight.device).view(CODES)
    scales = torch.empty((_blocks(n), _blocks(k)), dtype=SCALES, device=weight.device)
    _lib.call("ldb_pack_weight_fp8", _stream(weight), weight.data_ptr(), ld, _DT[weight.dtype], codes.data_ptr(),
              codes.shape[1], scales.data_ptr(), scales.shape[1], n, k)
    return Fp8Weight(codes[:, :k], scales)


def matmul_fp8(a: Fp8Rows, w: Fp8Weight, bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
               act: int = _lib.LDB_ACT_NONE, out_dtype: torch.dtype = torch.float16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(a @ w^T + bias + residual)`` in ``out_dtype``, accumulated in FP32 and rounded once.

    ``a`` holds ``(..., K)`` rows, the result is ``(..., N)``; ``bias`` is
    float32 ``(N,)``, ``residual`` has the result's shape and dtype."""
    codes, scales, dev = a.codes, a.scales, a.codes.device
    if codes.dtype != CODES or w.codes.dtype != CODES or scales.dtype != SCALES or w.scales.dtype != SCALES:
        raise ValueError("matmul_fp8: codes must be float8_e4m3fn and scales float8_e8m0fnu")
    if codes.device.type != "cuda":
        raise ValueError("matmul_fp8: a must be on a CUDA device")
    if out_dtype not in _DT or (out is not None and out.dtype != out_dtype):
        raise ValueError("matmul_fp8: out_dtype must be float16, bfloat16 or float32, and out's dtype")
    m, k, a_ld = _flat(codes, "matmul_fp8: a")
    n, wk = w.codes.shape
    blocks = _blocks(k)
    lead = codes.shape[:-1]
    if wk != k:
        raise ValueError(f"matmul_fp8: rows of {k} channels times a weight of {wk}")
    if tuple(scales.shape) != (*lead, blocks) or tuple(w.scales.shape) != (_blocks(n), blocks):
        raise ValueError(f"matmul_fp8: scales {tuple(scales.shape)} and {tuple(w.scales.shape)} do not fit "
                         f"{tuple(codes.shape)} rows and a {(n, k)} weight")
    _, _, s_ld = _flat(scales, "matmul_fp8: scales")
    _, _, w_ld = _flat(w.codes, "matmul_fp8: weight")
    _, _, ws_ld = _flat(w.scales, "matmul_fp8: weight scales")
    if m <= 1:  # a single row: its stride is never used, but has to pass the alignment rule
        a_ld, s_ld = -(-a_ld // 16) * 16, -(-s_ld // 4) * 4
    if n == 1:
        w_ld = -(-w_ld // 16) * 16
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError(f"matmul_fp8: bias must be contiguous float32 ({n},)")
    if out is None:
        out = torch.empty((*lead, n), dtype=out_dtype, device=dev)
    elif tuple(out.shape) != (*lead, n):
        raise ValueError(f"matmul_fp8: out shape {tuple(out.shape)} != {(*lead, n)}")
    _, _, out_ld = _flat(out, "matmul_fp8: out")
    r_ld = 0
    if residual is not None:
        if residual.shape != out.shape or residual.dtype != out_dtype:
            raise ValueError(f"matmul_fp8: residual must be {out_dtype} {tuple(out.shape)}")
        _, _, r_ld = _flat(residual, "matmul_fp8: residual")
    for t in (scales, w.codes, w.scales, bias, residual, out):
        if t is not None and t.device != dev:
            raise ValueError("matmul_fp8: all tensors must be on one device")
    if m == 0:
        return out
    need = ctypes.c_size_t(0)
    _lib.call("ldb_matmul_fp8_workspace_size", m, n, k, ctypes.byref(need))
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
    with instrument.maybe_time("matmul_fp8", 2.0 * m * n * k):
        _lib.call("ldb_matmul_fp8", _stream(codes), codes.data_ptr(), a_ld, scales.data_ptr(), s_ld,
                  w.codes.data_ptr(), w_ld, w.scales.data_ptr(), ws_ld, _ptr(bias), _ptr(residual), r_ld,
                  out.data_ptr(), out_ld, m, n, k, act, _DT[out_dtype], _ptr(ws), need.value)
    return out
