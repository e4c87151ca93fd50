"""Paged 8- or 4-bit key/value cache: keys and values that are written once and read many times.

The 8-bit cache holds e4m3 codes in pages of tokens, ``(pages, kv_heads, page,
head_dim)`` for keys and for values, with one power-of-two scale (E8M0) per
page and head.  The 4-bit cache holds integers -8 .. 7, two to a byte, with one scale
for each 16 channels of a token: 9/16 of the bytes, and what is written is never
rounded again.  An item's tokens lie, in order, in the pages of its row of an
int32 page table, so items can share pages (several seeds of one text context)
and grow without moving.

    cache = KvCacheFp8.empty(pages, kv_heads, head_dim, page=64, device="cuda")    # or KvCacheInt4
    kv_append(cache, k, v, table, start)          # tokens start .. start + L of every item
    out = kv_attention(q, cache, table, lengths, scale=head_dim ** -0.5)
    k, v = kv_read(cache, table, lengths, tokens=77)              # as rows again

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
GROUP = 16  # channels per scale of the 4-bit cache

_current_device = torch._C._cuda_getDevice


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


class KvCacheInt4(NamedTuple):
    """uint8 codes ``k``, ``v`` ``(pages, kv_heads, page, head_dim / 2)``, the lower channel in a byte's low half,
    and scales ``(pages, kv_heads, head_dim / 16, page)``.

    A code ``c`` of 0 .. 15 stands for ``(c - 8) * s``; a scale byte for the
    float16 whose upper eight bits under the sign it is."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, *, page: int = 64,
              device: torch.device | str = "cuda") -> "KvCacheInt4":
        """An unwritten cache of ``pages`` pages of ``page`` tokens (16, 32, 64 or 128)."""
        if page not in PAGES or head_dim not in HEAD_DIMS:
            raise ValueError(f"pages hold {PAGES} tokens of {HEAD_DIMS} channels, got {page} of {head_dim}")
        shapes = [(pages, kv_heads, page, head_dim // 2)] * 2 + [(pages, kv_heads, head_dim // GROUP, page)] * 2
        return cls(*(torch.empty(s, dtype=torch.uint8, device=device) for s in shapes))


KvCache = KvCacheFp8 | KvCacheInt4


def _check_cache(cache: KvCache, name: str) -> tuple[tuple[int, ...], torch.device]:
    """((pages, kv_heads, page, head_dim), device)."""
    k, v, k_scale, v_scale = cache
    if isinstance(cache, KvCacheInt4):
        shape, device = k.shape, k.device
        if len(shape) != 4 or v.shape != shape or k.dtype != torch.uint8 or v.dtype != torch.uint8:
            raise ValueError(f"{name}: k and v must be uint8 (pages, kv_heads, page, head_dim / 2)")
        pages, heads, page, dim = shape[0], shape[1], shape[2], 2 * shape[3]
        if page not in PAGES or dim not in HEAD_DIMS:
            raise ValueError(f"{name}: pages hold {PAGES} tokens of {HEAD_DIMS} channels, got {page} of {dim}")
        per = (pages, heads, dim // GROUP, page)
        if (k_scale.shape != per or v_scale.shape != per or k_scale.dtype != torch.uint8
                or v_scale.dtype != torch.uint8):
            raise ValueError(f"{name}: scales must be uint8 {per}")
        if not k.is_cuda:
            raise ValueError(f"{name}: the cache must be on a CUDA device")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()
                and v.device == device and k_scale.device == device and v_scale.device == device):
            raise ValueError(f"{name}: the cache's tensors must be contiguous and on one device")
        return (pages, heads, page, dim), device
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


def _fields(cache: KvCache, table: torch.Tensor, per_item: torch.Tensor, name: str, what: str) -> tuple[tuple, int, int]:
    """The library's description of a cache and its table, the channels of a token, and the device's index.

    (All of it is looked at in one expression, as a token's call is bound by the host; what is wrong is found out after that.)"""
    k, v, k_scale, v_scale = cache
    shape, index = k.shape, k.get_device()
    if len(shape) == 4:
        pages, heads, page, dim = shape
        if isinstance(cache, KvCacheInt4):
            codes = scales = torch.uint8
            dim *= 2
            per = (pages, heads, dim // GROUP, page)
        else:
            codes, scales, per = CODES, SCALES, (pages, heads)
        if (page in PAGES and dim in HEAD_DIMS and index >= 0 and v.shape == shape and k_scale.shape == per
                and v_scale.shape == per and k.dtype is codes and v.dtype is codes and k_scale.dtype is scales
                and v_scale.dtype is scales and k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous()
                and v_scale.is_contiguous() and v.get_device() == index and k_scale.get_device() == index
                and v_scale.get_device() == index and per_item.ndim == 1 and table.ndim == 2
                and per_item.dtype is torch.int32 and table.dtype is torch.int32 and per_item.get_device() == index
                and table.get_device() == index and per_item.is_contiguous()):
            (batch,), (rows, width), (table_ld, step) = per_item.shape, table.shape, table.stride()
            if rows == batch and width and (step == 1 or width == 1):
                return ((k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), table.data_ptr(),
                         table_ld if batch > 1 else width, pages, heads, page, dim, width, batch), heads * dim, index)
    _, device = _check_cache(cache, name)
    if per_item.ndim != 1:
        raise ValueError(f"{name}: {what} must be one number per item")
    _check_table(table, per_item.shape[0], device, f"{name}: table")
    _check_index(per_item, 1, per_item.shape[0], device, f"{name}: {what}")
    raise ValueError(f"{name}: cache, table and {what} do not fit")


_APPEND, _READ, _ATTENTION = (_lib.DESCRIPTORS[f"ldb_kv_{n}_desc"] for n in ("append", "read", "attention"))


def kv_append(cache: KvCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, *,
              counts: torch.Tensor | None = None) -> None:
    """Write ``(B, L, kv_heads * head_dim)`` keys and values at positions ``start[b] ..`` of each item.

    Only the first ``counts[b]`` of item ``b``'s tokens where given (a causal
    ``kv_attention`` takes an item's last rows for its queries: see there).  What a
    page holds before ``start`` stays, in 8 bits rounded again if the page's scale has to
    grow for the new tokens (zeros and what is not finite never ask for that); anything at or after ``start`` in the touched
    pages counts as unwritten.  Items written together must not share the
    pages they write.  float16, bfloat16 or float32, any row and item stride.

    In 4 bits a value is within half its scale: a 15th of the largest of its 16
    channels and up to an eighth of that more (a scale has four bits), or up to 2^-18 more where that is
    greater (scales below 2^-14 lie 2^-17 apart).  Magnitudes past 6720
    saturate, below 2^-18 they vanish, and 16 channels with one that is not finite are NaN."""
    if isinstance(cache, KvCacheInt4):
        return _append_int4(cache, k, v, table, start, counts)
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


def _append_int4(cache: KvCacheInt4, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
                 counts: torch.Tensor | None) -> None:
    fields, channels, index = _fields(cache, table, start, "kv_append", "start")
    if index != _current_device():
        with torch.cuda.device(index):
            return _append_int4(cache, k, v, table, start, counts)
    dtype = _DT.get(k.dtype)
    if dtype is None or v.dtype != k.dtype:
        raise ValueError("kv_append: k and v must share dtype float16, bfloat16 or float32")
    shape = k.shape
    if len(shape) != 3 or v.shape != shape or shape[2] != channels or shape[0] != fields[-1]:
        raise ValueError(f"kv_append: k and v must be ({fields[-1]}, L, {channels}), got {tuple(shape)} and {tuple(v.shape)}")
    if k.get_device() != index or v.get_device() != index:
        raise ValueError("kv_append: k and v must be on the cache's device")
    (k_batch, k_ld, k_step), (v_batch, v_ld, v_step) = k.stride(), v.stride()
    if k_step != 1 or v_step != 1:
        raise ValueError("kv_append: channel axis must have unit stride")
    if counts is not None:
        _check_index(counts, 1, shape[0], k.device, "kv_append: counts")
    _launcher("kv_append")("ldb_kv_append_int4", _raw_stream(index), _lib.packed(
        "kv_append", _APPEND, dtype, *fields, k.data_ptr(), v.data_ptr(), k_ld, k_batch, v_ld, v_batch, start.data_ptr(),
        0 if counts is None else counts.data_ptr(), shape[1]))


def kv_attention(q: torch.Tensor, cache: KvCache, table: torch.Tensor, lengths: torch.Tensor, *, scale: float,
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
    they have pages.  Over 8 bits, a query's channels are exact down to 2^-10 (float16 2^-7) of
    its row's largest and within 2^-18 of that below, for up to 48 rows of a
    key/value head (queries times the heads that share it) down to 2^-14; weights
    are rounded to 11 bits down to 2^-29 of the row's largest, from 49 rows on at
    least to 2^-21, and lost below 2^-40 and 2^-32; scores (as powers of two: times scale log2(e)) are to stay below
    2^24, as weights overflow from there on.  Over 4 bits queries are exact (bfloat16
    down to 2^-31 of the row's largest); the weights have 11 bits down to 2^-25, from 49 rows on
    2^-21, and are lost below 2^-36 and 2^-32; scores may be as large as 2^127."""
    if isinstance(cache, KvCacheInt4):
        return _attention_int4(q, cache, table, lengths, scale, causal, out)
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


def _attention_int4(q: torch.Tensor, cache: KvCacheInt4, table: torch.Tensor, lengths: torch.Tensor, scale: float,
                    causal: bool, out: torch.Tensor | None) -> torch.Tensor:
    fields, row, index = _fields(cache, table, lengths, "kv_attention", "lengths")
    if index != _current_device():
        with torch.cuda.device(index):
            return _attention_int4(q, cache, table, lengths, scale, causal, out)
    kv_heads, page, dim, width, batch = fields[-5:]
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"kv_attention: queries must be float16 or bfloat16, got {q.dtype}")
    shape = q.shape
    if len(shape) != 3 or q.get_device() != index or shape[2] % row or shape[2] == 0 or shape[0] != batch:
        raise ValueError(f"kv_attention: queries must be ({batch}, L, n * {row}) on the cache's device, got {tuple(shape)}")
    _, queries, channels = shape
    q_batch, q_ld, q_step = q.stride()
    if q_step != 1:
        raise ValueError("kv_attention: channel axis must have unit stride")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_ld, out_batch = channels, queries * channels
    else:
        if out.shape != shape or out.dtype != q.dtype or out.get_device() != index or out.stride(2) != 1:
            raise ValueError("kv_attention: out must have q's shape, dtype and device, and unit channel stride")
        out_batch, out_ld, _ = out.stride()
    heads = channels // dim
    need = _workspace_bytes("ldb_kv_attention_int4_workspace_size", index, batch, queries, heads, kv_heads, dim,
                            width * page)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _launcher("kv_attention")("ldb_kv_attention_int4", _raw_stream(index), _lib.packed(
        "kv_attention", _ATTENTION, _DT[q.dtype], *fields, q.data_ptr(), out.data_ptr(), q_ld, q_batch, out_ld, out_batch,
        lengths.data_ptr(), 0 if ws is None else ws.data_ptr(), need, queries, heads, int(causal), scale))
    return out


def kv_read(cache: KvCache, table: torch.Tensor, lengths: torch.Tensor, *, tokens: int,
            start: torch.Tensor | None = None, dtype: torch.dtype = torch.float16,
            out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``(B, tokens, kv_heads * head_dim)`` of each item's tokens ``start[b] ..`` (from 0 without ``start``).

    Rows at or behind ``lengths[b]`` are zeros.  float16, bfloat16 or float32:
    exact from a 4-bit cache, rounded once from 8 bits.  ``out`` takes a pair of tensors to
    write, of any row and item stride."""
    fields, channels, index = _fields(cache, table, lengths, "kv_read", "lengths")
    if index != _current_device():
        with torch.cuda.device(index):
            return kv_read(cache, table, lengths, tokens=tokens, start=start, dtype=dtype, out=out)
    if not 0 <= tokens < 2 ** 31:
        raise ValueError(f"kv_read: tokens must be at least 0 and below 2^31, got {tokens}")
    batch = fields[-1]
    if start is not None:
        _check_index(start, 1, batch, lengths.device, "kv_read: start")
    shape = (batch, tokens, channels)
    if out is None:
        if dtype not in _DT:
            raise ValueError(f"kv_read: dtype must be float16, bfloat16 or float32, got {dtype}")
        k_batch = v_batch = tokens * channels
        k_ld = v_ld = channels
        # (3.0 us of the host's; new_empty twice 4.2)
        k = torch.empty_strided(shape, (k_batch, k_ld, 1), dtype=dtype, device=cache[0].device)
        v = torch.empty_like(k)
    else:
        k, v = out
        if (k.shape != shape or v.shape != shape or k.dtype not in _DT or v.dtype != k.dtype or k.get_device() != index
                or v.get_device() != index):
            raise ValueError(f"kv_read: out must be two tensors {shape} of one float dtype on the cache's device")
        (k_batch, k_ld, k_step), (v_batch, v_ld, v_step) = k.stride(), v.stride()
        if k_step != 1 or v_step != 1:
            raise ValueError("kv_read: channel axis must have unit stride")
    _launcher("kv_read")("ldb_kv_read_int4" if isinstance(cache, KvCacheInt4) else "ldb_kv_read_fp8", _raw_stream(index),
            _lib.packed("kv_read", _READ, _DT[k.dtype], *fields, k.data_ptr(), v.data_ptr(), k_ld, k_batch, v_ld, v_batch,
                       lengths.data_ptr(), 0 if start is None else start.data_ptr(), tokens))
    return k, v
