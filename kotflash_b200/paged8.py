# SPDX-License-Identifier: Apache-2.0
"""Paged KV cache in 8 bits: half the bytes of ``PagedKVCache``, the same tables.

K and V rows are stored as 8-bit codes, ``torch.float8_e4m3fn`` or
``torch.int8``, with a power of two as the scale of each block of tokens and
head (``torch.float8_e8m0fnu``, one byte).  The block is one token by default;
scales [pages, Hkv, page_size / block] say what it is.

* ``append_paged_kv8``: 16-bit K/V rows to their slots, rounded to codes;
* ``read_paged_kv8``: rows of given slots back in 16 bits;
* ``paged_attention8``: one new token per request over its pages, with the
  append of that token's own row fused in on request;
* ``PagedKVCache8``: pools, scales and tables, and these calls on them.

What a row stands for.  A block's scale is the smallest power of two with which
its largest magnitude is at most 448 (e4m3) or rounds to at most 127 (int8),
within 2^-60 and 2^60; codes are rounded to nearest, ties to even.  So an
element is off by at most 2^-4 of itself or 2^-10 of the scale, whichever is
larger (e4m3), or by half of the scale (int8; above the smallest scale that is
less than 1 / 127.5 of its block's largest).  With several tokens to a scale,
rows stored before it grew were rounded again each time: they are off by less
than 2^-4 of the element and 2^-9 of the scale together (e4m3), or by less than
the scale (int8).  Blocks with an infinity, a NaN or a magnitude that no scale holds stand for NaN
as a whole.  What the codes stand for is exact in bf16 and, within its range,
in fp16.

fp16 and bf16 rows, head dims that are multiples of 8 in [16, 128], on an
sm_100 device through ``libkotflash_b200.so``; nothing falls back to another
implementation.  Inference only.  The reference has neither pages nor 8 bits.
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional, Tuple, Union

import torch

from . import _ext
from .paged import PagedKVCache, _check_device, _check_inference, _check_int32, _check_slots, _check_table

_DTYPES = {torch.float16: _ext.KF_F16, torch.bfloat16: _ext.KF_BF16}
_FORMATS = {torch.float8_e4m3fn: _ext.KF_E4M3, torch.int8: _ext.KF_INT8}
_SCALES = torch.float8_e8m0fnu
_INT32, _INT64 = torch.int32, torch.int64
_CONTIGUOUS = torch.contiguous_format
_pack_append, _pack_decode, _pack_step = _ext.pack_paged8_append, _ext.pack_paged8_decode, _ext.pack_paged8_step
_raw_stream, _is_sm100, _status_ptr = _ext.raw_stream, _ext.is_sm100, _ext.status_ptr


# As in paged.py: a valid call is tested in one expression; these find out what
# to say when that is false.

def _check_cache(what: str, k_pages, v_pages, k_scales, v_scales) -> None:
    for t in (k_pages, v_pages, k_scales, v_scales):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: pages and scales must be torch.Tensor instances")
    if k_pages.dtype not in _FORMATS:
        raise TypeError(f"{what}: pages must be float8_e4m3fn or int8, got {k_pages.dtype}")
    if v_pages.dtype != k_pages.dtype:
        raise ValueError(f"{what}: K and V pages must have one dtype")
    if k_scales.dtype != _SCALES or v_scales.dtype != _SCALES:
        raise TypeError(f"{what}: scales must be float8_e8m0fnu")
    if k_pages.ndim != 4 or v_pages.ndim != 4:
        raise ValueError(f"{what}: expected 4-D pages in [pages, Hkv, page_size, D] layout")
    if k_pages.shape != v_pages.shape:
        raise ValueError(f"{what}: K/V page shapes must match")
    if k_scales.ndim != 3 or k_scales.shape != v_scales.shape or k_scales.shape[:2] != k_pages.shape[:2]:
        raise ValueError(f"{what}: scales must be [pages, Hkv, page_size / block]")
    page_size, blocks = k_pages.shape[2], k_scales.shape[2]
    if blocks == 0 or page_size % blocks:
        raise ValueError(f"{what}: scales must be [pages, Hkv, page_size / block]")
    if blocks > 1 and (k_scales.stride(2) != 1 or v_scales.stride(2) != 1):
        raise ValueError(f"{what}: the scales of a page and head must be contiguous")


def _check_rows(what: str, rows) -> None:
    for t in rows:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: queries and K/V rows must be torch.Tensor instances")
    for t in rows:
        if t.dtype not in _DTYPES:
            raise TypeError(f"{what} supports float16 and bfloat16 rows, got {t.dtype}")
        if t.dtype != rows[0].dtype:
            raise ValueError(f"{what}: dtypes must match")
        if t.ndim != 4:
            raise ValueError(f"{what}: expected 4-D tensors")


def _cache(index, k_pages, v_pages, k_scales, v_scales):
    """The fields of a kf_paged8_cache on device ``index``, or None where
    ``_check_cache`` or ``_check_device`` would complain."""
    pages, hkv, page_size, d = ks = k_pages.shape
    n, h, blocks = ss = k_scales.shape
    (k0, k1, k2), (v0, v1, v2) = k_scales.stride(), v_scales.stride()
    dtype = k_pages.dtype
    if (index < 0 or k_pages.get_device() != index or v_pages.get_device() != index or k_scales.get_device() != index
            or v_scales.get_device() != index or not _is_sm100(index) or dtype not in _FORMATS
            or v_pages.dtype is not dtype or k_scales.dtype is not _SCALES or v_scales.dtype is not _SCALES
            or v_pages.shape != ks or n != pages or h != hkv or blocks == 0 or page_size % blocks
            or v_scales.shape != ss or (blocks > 1 and (k2 != 1 or v2 != 1))):
        return None
    return (k_pages.data_ptr(), pages, hkv, page_size, d, *k_pages.stride(), v_pages.data_ptr(), pages, hkv, page_size, d,
            *v_pages.stride(), k_scales.data_ptr(), v_scales.data_ptr(), k0, k1, v0, v1, page_size // blocks,
            _FORMATS[dtype])


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it, with contiguous rows on 16 bytes."""
    good = t.data_ptr() % 16 == 0 and t.stride(3) == 1 and all(
        t.shape[i] == 1 or t.stride(i) % 8 == 0 for i in range(3))
    return t if good else t.clone(memory_format=_CONTIGUOUS)


def append_paged_kv8(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    new_k: torch.Tensor,
    new_v: torch.Tensor,
    slots: torch.Tensor,
) -> None:
    """Store 16-bit K/V rows in the pages of an 8-bit pool.

    new_k and new_v are [N, Hkv, S, D] with any strides; token t = n * S + s
    goes to slot slots[t] (int64 [N * S]), row slots[t] % page_size of page
    slots[t] // page_size.  Tokens whose slot is outside the pool (-1) are
    skipped; no two tokens share a slot; N or S may be 0.  k_scales and v_scales are [pages, Hkv, page_size
    / block], block a power of two up to 128.

    With more than one token to a scale, a call's rows of one block share its
    scale, wherever their tokens stand in slots.  If the block's first row is
    not among them, they join the rows before the first of them: if the scale
    has to grow, those rows' codes are rounded again (a scale never shrinks
    while its block lasts).  The first row of a block begins it anew.  Rows
    behind the first written one that the call does not write keep their codes
    and take the new scale: write them before they are read.
    """
    what = "append_paged_kv8"
    try:
        index = k_pages.get_device()
        ns = new_k.shape
        cache = _cache(index, k_pages, v_pages, k_scales, v_scales)
        good = (
            cache is not None and new_k.dtype in _DTYPES
            and new_v.dtype is new_k.dtype and new_k.get_device() == index and new_v.get_device() == index
            and slots.get_device() == index and slots.dtype is _INT64 and len(ns) == 4 and new_v.dim() == 4
            and slots.shape == (ns[0] * ns[2],) and slots.is_contiguous()
            and not (torch.is_grad_enabled() and (new_k.requires_grad or new_v.requires_grad)))
    except (AttributeError, TypeError, ValueError, RuntimeError):
        good = False
    if not good:
        _check_cache(what, k_pages, v_pages, k_scales, v_scales)
        _check_rows(what, (new_k, new_v))
        _check_slots(what, slots, new_k.shape[0] * new_k.shape[2], "one slot for each new K/V row")
        _check_inference(what, new_k, new_v)
        _check_device(what, k_pages, v_pages, k_scales, v_scales, new_k, new_v, slots)
        raise RuntimeError(f"{what}: invalid arguments")
    if new_v.shape != ns:
        raise ValueError(f"{what}: new K/V shapes must match")
    if ns[1] != k_pages.shape[1] or ns[3] != k_pages.shape[3]:
        raise ValueError(f"{what}: new K/V heads and head_dim must match the pages")
    if ns[0] == 0 or ns[2] == 0:  # a step that admits no prompt
        return
    new_k, new_v = _aligned(new_k), _aligned(new_v)
    rc = _ext.load().kf_paged8_append(_pack_append(
        *cache, new_k.data_ptr(), *ns, *new_k.stride(), new_v.data_ptr(), *ns, *new_v.stride(), slots.data_ptr(), _DTYPES[new_k.dtype], _raw_stream(index)))
    if rc:
        _ext.check(rc, "kf_paged8_append")


def read_paged_kv8(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    slots: torch.Tensor,
    *,
    dtype: torch.dtype,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V rows of the given slots (int64 [T]) as [1, Hkv, T, D] in dtype.

    What the codes stand for, rounded where dtype cannot hold it (only fp16, at
    the ends of its range).  Rows whose slot is outside the pool (-1) are 0.
    """
    what = "read_paged_kv8"
    if dtype not in _DTYPES:
        raise TypeError(f"{what} supports float16 and bfloat16, got {dtype}")
    try:
        index = k_pages.get_device()
        cache = _cache(index, k_pages, v_pages, k_scales, v_scales)
        good = (cache is not None and slots.get_device() == index
                and slots.dtype is _INT64 and slots.dim() == 1 and slots.is_contiguous())
    except (AttributeError, TypeError, ValueError, RuntimeError):
        good = False
    if not good:
        _check_cache(what, k_pages, v_pages, k_scales, v_scales)
        _check_slots(what, slots, slots.numel() if isinstance(slots, torch.Tensor) else 0, "[tokens]")
        _check_device(what, k_pages, v_pages, k_scales, v_scales, slots)
        raise RuntimeError(f"{what}: invalid arguments")
    _, hkv, _, d = k_pages.shape
    tokens = slots.shape[0]
    k = slots.new_empty((1, hkv, tokens, d), dtype=dtype)
    v = torch.empty_like(k)
    if tokens == 0:
        return k, v
    rows = (1, hkv, tokens, d, hkv * tokens * d, tokens * d, d, 1)
    rc = _ext.load().kf_paged8_read(_pack_append(
        *cache, k.data_ptr(), *rows, v.data_ptr(), *rows, slots.data_ptr(), _DTYPES[dtype], _raw_stream(index)))
    if rc:
        _ext.check(rc, "kf_paged8_read")
    return k, v


def _check_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, new_k, new_v, slots) -> None:
    what = "paged_attention8"
    if (new_k is None) != (new_v is None) or (new_k is None) != (slots is None):
        raise ValueError(f"{what}: new_k, new_v and slots go together")
    rows = () if new_k is None else (new_k, new_v)
    _check_cache(what, k_pages, v_pages, k_scales, v_scales)
    _check_rows(what, (q, *rows))
    _check_int32(what, block_table=block_table, lengths=lengths)
    b, hq = q.shape[:2]
    hkv = k_pages.shape[1]
    _check_table(what, block_table, b)
    if lengths.ndim != 1 or lengths.shape[0] != b or not lengths.is_contiguous():
        raise ValueError(f"{what}: lengths must be a contiguous [requests] tensor")
    if rows:
        _check_slots(what, slots, b, "one for each request")
    if b == 0 or hq == 0 or hkv == 0:
        raise ValueError(f"{what}: batch and head dimensions must be non-zero")
    if hq % hkv:
        raise ValueError("num_query_heads must be divisible by num_kv_heads (GQA/MQA)")
    _check_inference(what, q, *rows)
    _check_device(what, q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, *rows, *((slots,) if rows else ()))


@lru_cache(maxsize=256)
def _workspace_elements(hq: int, hkv: int, d: int, device_index: int) -> int:
    """Workspace of kf_paged8_decode in 16-bit elements."""
    return _ext.load().kf_paged8_decode_workspace_bytes(hq, hkv, d, _ext.sm_count(device_index)) // 2 + 8


def paged_attention8(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: Optional[float] = None,
    new_k: Optional[torch.Tensor] = None,
    new_v: Optional[torch.Tensor] = None,
    slots: Optional[torch.Tensor] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``paged_attention`` over an 8-bit paged KV cache.

    q is [B, Hq, 1, D] in fp16 or bf16, rows contiguous and on 16 bytes like
    those of new_k and new_v; k_pages and v_pages [pages, Hkv,
    page_size, D] in float8_e4m3fn or int8, with any positive strides whose rows
    are contiguous and 16-byte aligned; k_scales and v_scales [pages, Hkv,
    page_size / block].  block_table, lengths, masking and results are those of
    ``paged_attention``, K and V being what their codes stand for.

    new_k and new_v [B, Hkv, 1, D] in q's dtype with slots append on the way:
    where slots[b] >= 0, the slot of position lengths[b] - 1, that position's
    row is stored as ``append_paged_kv8`` stores it and attended to as stored.
    With one token to a scale that happens in the same launch.
    """
    if scale is not None:
        try:
            scale = float(scale)
        except (TypeError, ValueError) as exc:
            raise TypeError("scale must be a finite real number or None") from exc
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
    try:
        index = q.get_device()
        dtype = q.dtype
        b, hq, _, d = qs = q.shape
        cache = _cache(index, k_pages, v_pages, k_scales, v_scales)
        hkv = k_pages.shape[1]
        requests, max_pages = block_table.shape
        row_stride, column_stride = block_table.stride()
        grad = torch.is_grad_enabled()
        good = (
            cache is not None and block_table.get_device() == index
            and lengths.get_device() == index and dtype in _DTYPES and block_table.dtype is _INT32
            and lengths.dtype is _INT32 and lengths.dim() == 1 and lengths.numel() == b and requests == b
            and column_stride == 1 and lengths.is_contiguous() and b > 0 and hq > 0 and hkv > 0 and hq % hkv == 0
            and not (grad and q.requires_grad))
        if new_k is not None or new_v is not None or slots is not None:
            good = good and (
                new_k.get_device() == index and new_v.get_device() == index and slots.get_device() == index
                and new_k.dtype is dtype and new_v.dtype is dtype and new_k.dim() == 4 and new_v.dim() == 4
                and slots.dtype is _INT64 and slots.dim() == 1 and slots.numel() == b and slots.is_contiguous()
                and not (grad and (new_k.requires_grad or new_v.requires_grad)))
    except (AttributeError, TypeError, ValueError, RuntimeError):
        good = False
    if not good:
        _check_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, new_k, new_v, slots)
        # all is well: a table of one column may have any stride
    if scale is None:
        scale = 1.0 / math.sqrt(d) if d else 1.0
    out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    elements = _workspace_elements(hq, hkv, d, index)
    workspace = q.new_empty(elements)
    if return_lse:
        lse = q.new_empty((b, hq, 1), dtype=torch.float32)
        lse_ptr = lse.data_ptr()
    else:
        lse_ptr = 0
    rest = (block_table.data_ptr(), max_pages, row_stride, lengths.data_ptr(), out.data_ptr(), lse_ptr, _DTYPES[dtype], scale,
            workspace.data_ptr(), elements * 2, _status_ptr(index), _raw_stream(index))
    if new_k is None:
        args = _pack_decode(*cache, q.data_ptr(), *qs, *q.stride(), *rest)
    else:
        args = _pack_step(*cache, q.data_ptr(), *qs, *q.stride(), new_k.data_ptr(), *new_k.shape, *new_k.stride(),
                          new_v.data_ptr(), *new_v.shape, *new_v.stride(), slots.data_ptr(), *rest)
    rc = _ext.load().kf_paged8_decode(args)
    if rc:
        _ext.check(rc, "kf_paged8_decode")
    return (out, lse) if return_lse else out


class PagedKVCache8(PagedKVCache):
    """``PagedKVCache`` whose pools hold 8-bit codes (``dtype``: float8_e4m3fn
    or int8) with a scale for each ``scale_block`` tokens and head.

    Rows go in and come back in fp16 or bf16; ``read`` gives those of slots
    back.  Everything else is as there.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, max_requests: int,
                 max_pages: int, *, layers: int = 1, scale_block: int = 1, device: Union[torch.device, str],
                 dtype: torch.dtype = torch.float8_e4m3fn) -> None:
        if dtype not in _FORMATS:
            raise TypeError(f"dtype must be float8_e4m3fn or int8, got {dtype}")
        self._set_up(num_pages, page_size, kv_heads, head_dim, max_requests, max_pages, layers, device)
        if isinstance(scale_block, bool) or not isinstance(scale_block, int) or not 0 < scale_block <= 128 \
                or scale_block & (scale_block - 1) or page_size % scale_block:
            raise ValueError("scale_block must be a power of two up to 128 that divides page_size")
        # rows begin on 16 bytes
        shape = (layers, num_pages, kv_heads, page_size, -(-head_dim // 16) * 16)
        self.k = torch.empty(shape, device=device, dtype=dtype)[..., :head_dim]
        self.v = torch.empty(shape, device=device, dtype=dtype)[..., :head_dim]
        scales = (layers, num_pages, kv_heads, page_size // scale_block)
        self.k_scales = torch.zeros(scales, device=device, dtype=torch.uint8).view(_SCALES)
        self.v_scales = torch.zeros(scales, device=device, dtype=torch.uint8).view(_SCALES)

    def _layer(self, layer: int):
        return self.k[layer], self.v[layer], self.k_scales[layer], self.v_scales[layer]

    def append(self, new_k: torch.Tensor, new_v: torch.Tensor, slots: torch.Tensor, *, layer: int = 0) -> None:
        """Store K/V rows [N, Hkv, S, D] at the slots that ``reserve`` gave."""
        append_paged_kv8(*self._layer(layer), new_k, new_v, slots)

    def read(self, slots: torch.Tensor, *, dtype: torch.dtype, layer: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """The K and V rows at slots, [1, Hkv, len(slots), D] in dtype."""
        return read_paged_kv8(*self._layer(layer), slots, dtype=dtype)

    def attend(self, q: torch.Tensor, *, layer: int = 0, scale: Optional[float] = None,
               return_lse: bool = False):
        """One query token per request slot [max_requests, Hq, 1, D] over its pages."""
        return paged_attention8(q, *self._layer(layer), self.block_table, self.lengths, scale=scale,
                                return_lse=return_lse)

    def append_and_attend(self, q: torch.Tensor, new_k: torch.Tensor, new_v: torch.Tensor, slots: torch.Tensor, *,
                          layer: int = 0, scale: Optional[float] = None, return_lse: bool = False):
        """Store the newest K/V row of every request that has a slot and attend, as there."""
        return paged_attention8(q, *self._layer(layer), self.block_table, self.lengths, scale=scale, new_k=new_k,
                                new_v=new_v, slots=slots, return_lse=return_lse)
