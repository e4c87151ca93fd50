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
import functools
from typing import NamedTuple

import torch

from . import _lib, instrument
from .ops import _DT, _rows

BLOCK = 128  # channels per scale of a row; rows and channels per scale of a weight
CODES = torch.float8_e4m3fn
SCALES = torch.float8_e8m0fnu

# The current stream's handle by device index.  (A single token's call is
# bound by the host: building a torch.cuda.Stream to read its handle takes longer than a launch.)
_raw_stream = torch._C._cuda_getCurrentRawStream

_MAX_ROWS = 2 ** 31 - 1  # the library counts rows in 32 bits


class Fp8Rows(NamedTuple):
    """``(..., K)`` e4m3 codes and ``(..., ceil(K / 128))`` E8M0 scales.

    Code rows are 16-byte aligned (row stride a multiple of 16), scale rows
    4-byte aligned (row stride a multiple of 4)."""

    codes: torch.Tensor
    scales: torch.Tensor


class Fp8Weight(NamedTuple):
    """``(N, K)`` e4m3 codes (row stride a multiple of 16) and ``(ceil(N / 128), ceil(K / 128))`` E8M0 scales."""

    codes: torch.Tensor
    scales: torch.Tensor


def _flat(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, channels, row stride) of a channels-last tensor dense over its rows."""
    shape = t.shape
    if len(shape) < 2:
        raise ValueError(f"{name}: expected (..., channels) with at least two axes")
    k = shape[-1]
    if t.is_contiguous() and k:
        rows, ld = t.numel() // k, k
    elif len(shape) == 2:
        rows = shape[0]
        ld, step = t.stride()
        if step != 1 and k != 1:
            raise ValueError(f"{name}: channel axis must have unit stride")
    else:
        per, k, ld = _rows(t)
        rows = shape[0] * per
        if shape[0] > 1 and per and t.stride(0) != per * ld:
            raise ValueError(f"{name}: tensor must be dense over its rows")
    if rows > _MAX_ROWS:
        raise ValueError(f"{name}: {rows} rows (at most {_MAX_ROWS})")
    return rows, k, max(ld, k) if rows <= 1 else ld


def _quantized(x: torch.Tensor, k: int) -> tuple[Fp8Rows, int, int]:
    """Unwritten rows for ``x``'s leading axes and ``k`` channels, and their strides."""
    lead = x.shape[:-1]
    blocks = (k + 127) // 128
    ld, s_ld = (k + 15) // 16 * 16, (blocks + 3) // 4 * 4
    per_row, rows = [], 1  # rows between neighbours of each leading axis
    for n in reversed(lead):
        per_row.insert(0, rows)
        rows *= n
    if ld == k:
        codes = torch.empty_like(x, dtype=CODES, memory_format=torch.contiguous_format)
    else:  # (the padding behind the last row too)
        codes = x.new_empty(rows * ld, dtype=CODES).as_strided((*lead, k), [n * ld for n in per_row] + [1])
    scales = x.new_empty_strided((*lead, blocks), [n * s_ld for n in per_row] + [1], dtype=SCALES)
    return Fp8Rows(codes, scales), ld, s_ld


def _launcher(kind: str, flops: float = 0.0):
    """``_lib.call``, inside the active timer's measurement if there is one.

    (A context manager around every call costs a tenth of a single token's.)"""
    if instrument.active() is None:
        return _lib.call

    def call(name: str, *args) -> None:
        with instrument.maybe_time(kind, flops):
            _lib.call(name, *args)

    return call


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(name: str, device: int, *sizes: int) -> int:
    """What the library's ``name`` says for these sizes (asking costs a token's call a tenth of its time)."""
    need = ctypes.c_size_t()
    _lib.call(name, *sizes, ctypes.byref(need))
    return need.value


def _check_input(x: torch.Tensor, name: str) -> None:
    if x.dtype not in _DT:
        raise ValueError(f"{name} must be float16, bfloat16 or float32, got {x.dtype}")
    if not x.is_cuda:
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
    h = residual_ptr = h_ptr = None
    r_ld = 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError("rms_norm_fp8: residual must have x's shape, dtype and device")
        r_ld = _flat(residual, "rms_norm_fp8: residual")[2]
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
        residual_ptr, h_ptr = residual.data_ptr(), h.data_ptr()
    out, ld, s_ld = _quantized(x, c)
    _launcher("rms_norm_fp8")("ldb_rms_norm_fp8", _raw_stream(x.get_device()), x.data_ptr(), x_ld, residual_ptr,
            r_ld, _DT[x.dtype], None if gamma is None else gamma.data_ptr(), eps, h_ptr, c, out.codes.data_ptr(), ld,
            out.scales.data_ptr(), s_ld, rows, c)
    return out, x if h is None else h


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """8-bit rows of ``(..., K)`` float16 / bfloat16 / float32 ``x`` (up to 32768 channels)."""
    _check_input(x, "quantize_rows: x")
    rows, k, x_ld = _flat(x, "quantize_rows: x")
    out, ld, s_ld = _quantized(x, k)
    _launcher("quantize_rows")("ldb_quantize_fp8_rows", _raw_stream(x.get_device()), x.data_ptr(), x_ld,
            _DT[x.dtype], out.codes.data_ptr(), ld, out.scales.data_ptr(), s_ld, rows, k)
    return out


def pack_weight_fp8(weight: torch.Tensor) -> Fp8Weight:
    """8-bit form of an ``(N, K)`` float16 / bfloat16 / float32 dense weight (once per weight)."""
    _check_input(weight, "pack_weight_fp8: weight")
    if weight.ndim != 2 or 0 in weight.shape:
        raise ValueError(f"pack_weight_fp8: expected an (N, K) weight, got {tuple(weight.shape)}")
    n, k, ld = _flat(weight, "pack_weight_fp8: weight")
    codes = torch.zeros((n, (k + 15) // 16 * 16), dtype=torch.uint8, device=weight.device).view(CODES)
    scales = torch.empty(((n + 127) // 128, (k + 127) // 128), dtype=SCALES, device=weight.device)
    _lib.call("ldb_pack_weight_fp8", _raw_stream(weight.get_device()), weight.data_ptr(), ld, _DT[weight.dtype],
              codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], n, k)
    return Fp8Weight(codes[:, :k], scales)


def matmul_fp8(a: Fp8Rows, w: Fp8Weight, bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
               act: int = _lib.LDB_ACT_NONE, out_dtype: torch.dtype = torch.float16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(a @ w^T + bias + residual)`` in ``out_dtype``, accumulated in FP32 and rounded once.

    ``a`` holds ``(..., K)`` rows, the result is ``(..., N)``; ``bias`` is
    float32 ``(N,)``, ``residual`` has the result's shape and dtype."""
    codes, scales = a
    w_codes, w_scales = w
    if codes.dtype != CODES or w_codes.dtype != CODES or scales.dtype != SCALES or w_scales.dtype != SCALES:
        raise ValueError("matmul_fp8: codes must be float8_e4m3fn and scales float8_e8m0fnu")
    if not codes.is_cuda:
        raise ValueError("matmul_fp8: a must be on a CUDA device")
    if out_dtype not in _DT or (out is not None and out.dtype != out_dtype):
        raise ValueError("matmul_fp8: out_dtype must be float16, bfloat16 or float32, and out's dtype")
    m, k, a_ld = _flat(codes, "matmul_fp8: a")
    n, wk, w_ld = _flat(w_codes, "matmul_fp8: weight")
    if wk != k or w_codes.ndim != 2:
        raise ValueError(f"matmul_fp8: rows of {k} channels times a weight of {tuple(w_codes.shape)}")
    s_rows, blocks, s_ld = _flat(scales, "matmul_fp8: scales")
    ws_rows, w_blocks, ws_ld = _flat(w_scales, "matmul_fp8: weight scales")
    lead = codes.shape[:-1]
    if (blocks != (k + 127) // 128 or w_blocks != blocks or scales.shape[:-1] != lead or w_scales.ndim != 2
            or ws_rows != (n + 127) // 128):
        raise ValueError(f"matmul_fp8: scales {tuple(scales.shape)} and {tuple(w_scales.shape)} do not fit "
                         f"{tuple(codes.shape)} rows and a {(n, k)} weight")
    if m <= 1:  # a single row: its stride is never used, but has to pass the alignment rule
        a_ld, s_ld = (a_ld + 15) // 16 * 16, (s_ld + 3) // 4 * 4
    if n == 1:
        w_ld = (w_ld + 15) // 16 * 16
    dev = codes.device
    bias_ptr = residual_ptr = ws_ptr = None
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous() or bias.device != dev:
            raise ValueError(f"matmul_fp8: bias must be contiguous float32 ({n},) on a's device")
        bias_ptr = bias.data_ptr()
    if out is None:
        out = codes.new_empty((*lead, n), dtype=out_dtype)
        out_ld = n
    else:
        if out.shape != (*lead, n):
            raise ValueError(f"matmul_fp8: out shape {tuple(out.shape)} != {(*lead, n)}")
        out_ld = _flat(out, "matmul_fp8: out")[2]
    r_ld = 0
    if residual is not None:
        if residual.shape != out.shape or residual.dtype != out_dtype or residual.device != dev:
            raise ValueError(f"matmul_fp8: residual must be {out_dtype} {tuple(out.shape)} on a's device")
        r_ld = _flat(residual, "matmul_fp8: residual")[2]
        residual_ptr = residual.data_ptr()
    if scales.device != dev or w_codes.device != dev or w_scales.device != dev or out.device != dev:
        raise ValueError("matmul_fp8: all tensors must be on one device")
    if m == 0:
        return out
    device = codes.get_device()
    need = _workspace_bytes("ldb_matmul_fp8_workspace_size", device, m, n, k)
    if need:
        ws = codes.new_empty(need, dtype=torch.uint8)
        ws_ptr = ws.data_ptr()
    _launcher("matmul_fp8", 2.0 * m * n * k)("ldb_matmul_fp8", _raw_stream(device), codes.data_ptr(), a_ld,
            scales.data_ptr(), s_ld, w_codes.data_ptr(), w_ld, w_scales.data_ptr(), ws_ld, bias_ptr, residual_ptr,
            r_ld, out.data_ptr(), out_ld, m, n, k, act, _DT[out_dtype], ws_ptr, need)
    return out
