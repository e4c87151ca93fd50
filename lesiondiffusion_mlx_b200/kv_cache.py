"""Paged 8-bit key/value cache: keys and values that are written once and read many times.

The cache holds e4m3 codes in pages of tokens, ``(pages, kv_heads, page,
head_dim)`` for keys and for values, with one power-of-two scale (E8M0) per
page and head.  An item's tokens lie, in order, in the pages of its row of an
int32 page table, so items can share pages (several seeds of one text context)
and grow without moving.

    cache = KvCacheFp8.empty(pages, kv_heads, head_dim, page=64, device="cuda")
    kv_append(cache, k, v, table, start)          # tokens start .. start + L of every item
    out = kv_attention(q, cache, table, lengths, scale=head_dim ** -0.5)

Lengths and positions are device tensors; a page number or a length outside
the cache is left out and sets the device status (``ldb_device_status``).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .fp8 import CODES, SCALES, _launcher, _raw_stream, _workspace_bytes
from .ops import _DT

HEAD_DIMS = (32, 64, 128)
PAGES = (16, 32, 64, 128)


class KvCacheFp8(NamedTuple):
    """Codes ``k``, ``v`` ``(pages, kv_heads, page, head_dim)`` and scales ``(pages, kv_heads)``."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, *, page: int = 64,
              device: torch.device | str = "cuda") -> "KvCacheFp8":
        """An unwritten cache of ``pages`` pages of ``page`` tokens (16, 32, 64 or 128)."""
        if page not in PAGES or head_dim not in HEAD_DIMS:
            raise ValueError(f"pages hold {PAGES} tokens of {HEAD_DIMS} channels, got {page} of {head_dim}")
        codes = [torch.empty((pages, kv_heads, page, head_dim), dtype=CODES, device=device) for _ in range(2)]
        scales = [torch.empty((pages, kv_heads), dtype=SCALES, device=device) for _ in range(2)]
        return cls(*codes, *scales)


def _check_cache(cache: KvCacheFp8, name: str) -> tuple[torch.Size, torch.device]:
    k, v, k_scale, v_scale = cache
    shape, device = k.shape, k.device
    if len(shape) != 4 or v.shape != shape or k.dtype != CODES or v.dtype != CODES:
        raise ValueError(f"{name}: k and v must be float8_e4m3fn (pages, kv_heads, page, head_dim)")
    if shape[2] not in PAGES or shape[3] not in HEAD_DIMS:
        raise ValueError(f"{name}: pages hold {PAGES} tokens of {HEAD_DIMS} channels, got {shape[2]} of {shape[3]}")
    if (k_scale.shape != shape[:2] or v_scale.shape != shape[:2] or k_scale.dtype != SCALES
            or v_scale.dtype != SCALES):
        raise ValueError(f"{name}: scales must be float8_e8m0fnu {tuple(shape[:2])}")
    if not k.is_cuda:
        raise ValueError(f"{name}: the cache must be on a CUDA device")
    if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()
            and v.device == device and k_scale.device == device and v_scale.device == device):
        raise ValueError(f"{name}: the cache's tensors must be contiguous and on one device")
    return shape, device


def _check_index(t: torch.Tensor, ndim: int, batch: int, device: torch.device, name: str) -> None:
    if t.dtype != torch.int32 or t.ndim != ndim or t.shape[0] != batch or t.device != device:
        raise ValueError(f"{name} must be an int32 {ndim}-axis tensor of {batch} items on the cache's device")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have unit stride along its last axis")


def _check_table(table: torch.Tensor, batch: int, device: torch.device, name: str) -> tuple[int, int]:
    """(columns, row stride) of the page table."""
    _check_index(table, 2, batch, device, name)
    width = table.shape[1]
    if width == 0:
        raise ValueError(f"{name} has no columns")
    return width, table.stride(0) if batch > 1 else width


def kv_append(cache: KvCacheFp8, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, *,
              counts: torch.Tensor | None = None) -> None:
    """Write ``(B, L, kv_heads * head_dim)`` keys and values at positions ``start[b] ..`` of each item.

    Only the first ``counts[b]`` of item ``b``'s tokens where given (a causal
    ``kv_attention`` takes an item's last rows for its queries: see there).  What a
    page holds before ``start`` stays, rounded again if the page's scale has to
    grow for the new tokens (zeros and what is not finite never ask for that); anything at or after ``start`` in the touched
    pages counts as unwritten.  Items written together must not share the
    pages they write.  float16, bfloat16 or float32, any row and item stride."""
    (pages, heads, page, dim), device = _check_cache(cache, "kv_append")
    if k.dtype not in _DT or v.dtype != k.dtype:
        raise ValueError("kv_append: k and v must share dtype float16, bfloat16 or float32")
    if k.ndim != 3 or v.shape != k.shape or k.shape[2] != heads * dim:
        raise ValueError(f"kv_append: k and v must be (B, L, {heads * dim}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.device != device or v.device != device:
        raise ValueError("kv_append: k and v must be on the cache's device")
    (k_batch, k_ld, k_step), (v_batch, v_ld, v_step) = k.stride(), v.stride()
    if k_step != 1 or v_step != 1:
        raise ValueError("kv_append: channel axis must have unit stride")
    batch, tokens, _ = k.shape
    width, table_ld = _check_table(table, batch, device, "kv_append: table")
    _check_index(start, 1, batch, device, "kv_append: start")
    if counts is not None:
        _check_index(counts, 1, batch, device, "kv_append: counts")
    _launcher("kv_append")("ldb_kv_append_fp8", _raw_stream(k.get_device()), k.data_ptr(), k_ld, k_batch,
            v.data_ptr(), v_ld, v_batch, _DT[k.dtype], cache.k.data_ptr(), cache.v.data_ptr(),
            cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages, heads, page, dim, table.data_ptr(), table_ld,
            width, start.data_ptr(), None if counts is None else counts.data_ptr(), batch, tokens)


def kv_attention(q: torch.Tensor, cache: KvCacheFp8, table: torch.Tensor, lengths: torch.Tensor, *, scale: float,
                 causal: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(q k^T * scale) v`` of ``(B, L, heads * head_dim)`` queries over each item's cached tokens.

    ``heads`` is a multiple of the cache's; query head ``h`` reads key/value
    head ``h // (heads / kv_heads)``.  Item ``b`` has ``lengths[b]`` tokens (0
    included).  With ``causal`` the queries are the item's last ``L`` tokens:
    query ``i`` sees the keys up to ``lengths[b] - L + i``.  (So an item that was
    given fewer than ``L`` tokens has its queries in the last rows, not in the
    first, where ``kv_append`` takes its tokens from: move them there, or attend to
    it by itself.)  A query that sees no key gives zeros; a NaN among the keys or
    values a query does not see does not reach it.  float16 or bfloat16, any row
    and item stride.

    The work is shared out by the table's columns, as the lengths are on the
    device: hand over ``table[:, :n]`` where the items hold far fewer tokens than
    they have pages.  A query's channels are exact down to 2^-10 (float16 2^-7) of
    its row's largest and within 2^-18 of that below, for up to 48 rows of a
    key/value head (queries times the heads that share it) down to 2^-14; weights
    are rounded to 11 bits down to 2^-29 of the row's largest, from 49 rows on at
    least to 2^-21, and lost below 2^-40 and 2^-32."""
    (pages, kv_heads, page, dim), device = _check_cache(cache, "kv_attention")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"kv_attention: queries must be float16 or bfloat16, got {q.dtype}")
    if q.ndim != 3 or q.device != device or q.shape[2] % (kv_heads * dim) or q.shape[2] == 0:
        raise ValueError(f"kv_attention: queries must be (B, L, n * {kv_heads * dim}) on the cache's device, got "
                         f"{tuple(q.shape)}")
    batch, queries, channels = q.shape
    q_batch, q_ld, q_step = q.stride()
    if q_step != 1:
        raise ValueError("kv_attention: channel axis must have unit stride")
    width, table_ld = _check_table(table, batch, device, "kv_attention: table")
    _check_index(lengths, 1, batch, device, "kv_attention: lengths")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or out.stride(2) != 1:
        raise ValueError("kv_attention: out must have q's shape, dtype and device, and unit channel stride")
    out_batch, out_ld, _ = out.stride()
    heads = channels // dim
    index = q.get_device()
    need = _workspace_bytes("ldb_kv_attention_fp8_table_workspace_size", index, batch, queries, heads, kv_heads, dim,
                            width * page)
    ws_ptr = None
    if need:
        ws = q.new_empty(need, dtype=torch.uint8)
        ws_ptr = ws.data_ptr()
    _launcher("kv_attention")("ldb_kv_attention_fp8", _raw_stream(index), q.data_ptr(), q_ld, q_batch,
            _DT[q.dtype], cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
            pages, kv_heads, page, dim, table.data_ptr(), table_ld, width, lengths.data_ptr(), out.data_ptr(), out_ld,
            out_batch, batch, queries, heads, scale, int(causal), ws_ptr, need)
    return out
