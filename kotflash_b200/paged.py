# SPDX-License-Identifier: Apache-2.0
"""Paged KV cache: many requests of different lengths in one pool of pages.

``PreallocatedKVCache`` gives every batch entry the same length and its full
capacity from the start.  Here the K and V rows of all requests lie in pools
``[pages, Hkv, page_size, D]``; a block table names each request's pages in
order, and the pages that nobody owns form a stack on the GPU.  Everything a
serving step needs is computed on the device from the device's own lengths,
so no call synchronises and a CUDA graph of a step follows the lengths:

* ``reserve_pages``: pages, table entries and slots for the tokens that each
  request brings;
* ``append_paged_kv``: K/V rows to their slots (prompts);
* ``paged_attention``: one new token per request over its pages, with the
  append of that token's own K/V row fused in on request (generation);
* ``release_pages``: the pages of finished requests back to the stack;
* ``PagedKVCache``: the pools, tables and stack, and these calls on them.

fp16 and bf16, head dims that are multiples of 8 in [16, 128], on an sm_100
device through ``libkotflash_b200.so``; nothing falls back to another
implementation.  Inference only.  The reference has no paging
(``kotflash/cache.py:91-98``).
"""
from __future__ import annotations

import math
from functools import lru_cache
from operator import index as _whole
from typing import Optional, Tuple, Union

import torch

from . import _ext

_DTYPES = {torch.float16: _ext.KF_F16, torch.bfloat16: _ext.KF_BF16}
_INT32, _INT64, _BOOL = torch.int32, torch.int64, torch.bool
_CONTIGUOUS = torch.contiguous_format
_pack_decode, _pack_step, _pack_append = _ext.pack_paged_decode, _ext.pack_paged_step, _ext.pack_paged_append
_pack_reserve, _pack_release = _ext.pack_paged_reserve, _ext.pack_paged_release
_raw_stream, _is_sm100, _status_ptr = _ext.raw_stream, _ext.is_sm100, _ext.status_ptr


# Each entry point below tests everything in one expression, which is what a
# valid call pays for (a few us of a call that lasts about ten); only when it
# is false do these functions find out what to say.

def _check_device(what: str, *tensors: torch.Tensor) -> None:
    """All tensors on one sm_100 device."""
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"{what} requires CUDA tensors on an sm_100 (B200) device")
    for t in tensors:
        if t.device != dev:
            raise ValueError(f"{what}: all tensors must be on the same device")
    if not _ext.is_sm100(dev.index):
        raise RuntimeError(f"{what} requires an sm_100 (B200) CUDA device")


def _check_pools(what: str, *tensors: torch.Tensor) -> None:
    """Pools and the K/V or query tensors beside them."""
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: K/V pages, K/V rows and queries must be torch.Tensor instances")
    for t in tensors:
        if t.dtype != tensors[0].dtype:
            raise ValueError(f"{what}: dtypes must match")
        if t.ndim != 4:
            raise ValueError(f"{what}: expected 4-D tensors, pages in [pages, Hkv, page_size, D] layout")
    if tensors[0].dtype not in _DTYPES:
        raise TypeError(f"{what} supports float16 and bfloat16, got {tensors[0].dtype}")


def _check_inference(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} is inference-only; disable gradients")


def _check_int32(what: str, **tensors: torch.Tensor) -> None:
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a torch.Tensor")
        if t.dtype != torch.int32:
            raise TypeError(f"{what}: {name} must be int32")


def _check_slots(what: str, slots: torch.Tensor, count: int, meaning: str) -> None:
    if not isinstance(slots, torch.Tensor):
        raise TypeError(f"{what}: slots must be a torch.Tensor")
    if slots.dtype != torch.int64:
        raise TypeError(f"{what}: slots must be int64")
    if slots.ndim != 1 or slots.shape[0] != count or not slots.is_contiguous():
        raise ValueError(f"{what}: slots must be contiguous, {meaning}")


def _check_table(what: str, block_table: torch.Tensor, requests: int) -> None:
    if block_table.ndim != 2 or block_table.shape[0] != requests:
        raise ValueError(f"{what}: block_table must be [requests, max_pages]")
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise ValueError(f"{what}: block_table rows must be contiguous")


def _check_attention(q, k_pages, v_pages, block_table, lengths, new_k, new_v, slots) -> None:
    what = "paged_attention"
    if (new_k is None) != (new_v is None) or (new_k is None) != (slots is None):
        raise ValueError(f"{what}: new_k, new_v and slots go together")
    rows = () if new_k is None else (new_k, new_v)
    _check_pools(what, q, k_pages, v_pages, *rows)
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
    _check_inference(what, q, k_pages, v_pages, *rows)
    _check_device(what, q, k_pages, v_pages, block_table, lengths, *rows, *((slots,) if rows else ()))


@lru_cache(maxsize=256)
def _workspace_elements(hq: int, hkv: int, d: int, device_index: int) -> int:
    """Workspace of kf_paged_decode in 16-bit elements."""
    return _ext.load().kf_paged_decode_workspace_bytes(hq, hkv, d, _ext.sm_count(device_index)) // 2 + 8


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: Optional[float] = None,
    new_k: Optional[torch.Tensor] = None,
    new_v: Optional[torch.Tensor] = None,
    slots: Optional[torch.Tensor] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of one new token per request over a paged KV cache.

    q is [B, Hq, 1, D]; k_pages and v_pages are [pages, Hkv, page_size, D]
    with any strides whose rows are contiguous and 16-byte aligned;
    block_table is int32 [B, max_pages] and lengths int32 [B].  Request b's
    token attends to positions 0 .. lengths[b] - 1, position p being row
    p % page_size of page block_table[b, p // page_size].  Positions whose
    table entry is not a page of the pool (-1, say) are masked,
    whatever the memory there holds.  A request that sees nothing yields 0 (LSE -inf).

    new_k and new_v [B, Hkv, 1, D] with slots (int64 [B]) append on the way:
    where slots[b] >= 0, the slot of position lengths[b] - 1, that position's
    row is new_k[b] / new_v[b], which is written to its page and attended to in
    the same launch (lengths already counts it, and no other request may read
    the slot); where slots[b] < 0 the request has no new row.  Returns [B, Hq, 1, D] in q's dtype and, with return_lse, the
    fp32 LSE [B, Hq, 1].
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
        _, hkv, _, _ = ks = k_pages.shape
        requests, max_pages = block_table.shape
        row_stride, column_stride = block_table.stride()
        grad = torch.is_grad_enabled()
        good = (
            index >= 0 and k_pages.get_device() == index and v_pages.get_device() == index
            and block_table.get_device() == index and lengths.get_device() == index and _is_sm100(index)
            and k_pages.dtype is dtype and v_pages.dtype is dtype and v_pages.dim() == 4
            and block_table.dtype is _INT32 and lengths.dtype is _INT32 and lengths.dim() == 1
            and lengths.numel() == b and requests == b and column_stride == 1 and lengths.is_contiguous()
            and b > 0 and hq > 0 and hkv > 0 and hq % hkv == 0
            and not (grad and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad))
        )
        if new_k is not None or new_v is not None or slots is not None:
            good = good and (
                new_k.get_device() == index and new_v.get_device() == index and slots.get_device() == index
                and new_k.dtype is dtype and new_v.dtype is dtype and new_k.dim() == 4 and new_v.dim() == 4
                and slots.dtype is _INT64 and slots.dim() == 1 and slots.numel() == b and slots.is_contiguous()
                and not (grad and (new_k.requires_grad or new_v.requires_grad)))
        code = _DTYPES.get(dtype, -1)
    except (AttributeError, TypeError, ValueError, RuntimeError):
        good = False
    if not good or code < 0:
        _check_attention(q, k_pages, v_pages, block_table, lengths, new_k, new_v, slots)
        # a table of one column may have any stride
        index, dtype, qs, ks = q.get_device(), q.dtype, q.shape, k_pages.shape
        b, hq, _, d = qs
        hkv, max_pages, row_stride, code = ks[1], block_table.shape[1], block_table.stride(0), _DTYPES[dtype]
    if scale is None:
        scale = 1.0 / math.sqrt(d) if d else 1.0
    lib = _ext.load()
    out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    elements = _workspace_elements(hq, hkv, d, index)
    workspace = q.new_empty(elements)
    if return_lse:
        lse = q.new_empty((b, hq, 1), dtype=torch.float32)
        lse_ptr = lse.data_ptr()
    else:
        lse_ptr = 0
    if new_k is None:
        args = _pack_decode(
            q.data_ptr(), *qs, *q.stride(), k_pages.data_ptr(), *ks, *k_pages.stride(),
            v_pages.data_ptr(), *v_pages.shape, *v_pages.stride(), block_table.data_ptr(), max_pages, row_stride,
            lengths.data_ptr(), out.data_ptr(), lse_ptr, code, scale, workspace.data_ptr(), elements * 2,
            _status_ptr(index), _raw_stream(index))
    else:
        args = _pack_step(
            q.data_ptr(), *qs, *q.stride(), k_pages.data_ptr(), *ks, *k_pages.stride(),
            v_pages.data_ptr(), *v_pages.shape, *v_pages.stride(), new_k.data_ptr(), *new_k.shape, *new_k.stride(),
            new_v.data_ptr(), *new_v.shape, *new_v.stride(), slots.data_ptr(), block_table.data_ptr(), max_pages,
            row_stride, lengths.data_ptr(), out.data_ptr(), lse_ptr, code, scale, workspace.data_ptr(), elements * 2,
            _status_ptr(index), _raw_stream(index))
    rc = lib.kf_paged_decode(args)
    if rc:
        _ext.check(rc, "kf_paged_decode")
    return (out, lse) if return_lse else out


def append_paged_kv(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    new_k: torch.Tensor,
    new_v: torch.Tensor,
    slots: torch.Tensor,
) -> None:
    """Copy K/V rows into the pages of a pool, bit for bit.

    new_k and new_v are [N, Hkv, S, D] with any strides; token t = n * S + s
    goes to slot slots[t] (int64 [N * S]), that is row slots[t] % page_size of
    page slots[t] // page_size.  Tokens whose slot is outside the pool (-1 for
    those that ``reserve_pages`` refused) are skipped; N or S may be 0.
    """
    try:
        index = k_pages.get_device()
        dtype = k_pages.dtype
        ns = new_k.shape
        good = (
            index >= 0 and _is_sm100(index) and dtype in _DTYPES and v_pages.dtype is dtype
            and new_k.dtype is dtype and new_v.dtype is dtype and slots.dtype is _INT64 and k_pages.ndim == 4
            and v_pages.ndim == 4 and len(ns) == 4 and new_v.ndim == 4 and slots.shape == (ns[0] * ns[2],)
            and slots.is_contiguous() and v_pages.get_device() == index and new_k.get_device() == index
            and new_v.get_device() == index and slots.get_device() == index
            and not (torch.is_grad_enabled() and (k_pages.requires_grad or v_pages.requires_grad
                                                  or new_k.requires_grad or new_v.requires_grad))
        )
    except (AttributeError, TypeError, RuntimeError):
        good = False
    if not good:
        what = "append_paged_kv"
        _check_pools(what, k_pages, v_pages, new_k, new_v)
        _check_slots(what, slots, new_k.shape[0] * new_k.shape[2], "one slot for each new K/V row")
        _check_inference(what, k_pages, v_pages, new_k, new_v)
        _check_device(what, k_pages, v_pages, new_k, new_v, slots)
        index, dtype, ns = k_pages.get_device(), k_pages.dtype, new_k.shape
    if ns[0] == 0 or ns[2] == 0:  # a step that admits no prompt
        if k_pages.shape != v_pages.shape:
            raise ValueError("append_paged_kv: K/V page shapes must match")
        if new_v.shape != ns:
            raise ValueError("append_paged_kv: new K/V shapes must match")
        if ns[1] != k_pages.shape[1] or ns[3] != k_pages.shape[3]:
            raise ValueError("append_paged_kv: new K/V heads and head_dim must match the pages")
        return
    rc = _ext.load().kf_paged_append(_pack_append(
        k_pages.data_ptr(), *k_pages.shape, *k_pages.stride(), v_pages.data_ptr(), *v_pages.shape, *v_pages.stride(),
        new_k.data_ptr(), *ns, *new_k.stride(), new_v.data_ptr(), *new_v.shape, *new_v.stride(),
        slots.data_ptr(), _DTYPES[dtype], _raw_stream(index),
    ))
    if rc:
        _ext.check(rc, "kf_paged_append")


def _tables_good(index, lengths, second, block_table, free_pages, free_count, lengths_out, free_count_out) -> bool:
    try:
        shape = lengths.shape
        return (
            index >= 0 and second.get_device() == index and block_table.get_device() == index
            and free_pages.get_device() == index and free_count.get_device() == index and _is_sm100(index)
            and lengths.dtype is _INT32 and block_table.dtype is _INT32 and free_pages.dtype is _INT32
            and free_count.dtype is _INT32 and lengths.dim() == 1 and second.shape == shape
            and block_table.dim() == 2 and block_table.shape[0] == shape[0] and block_table.stride(1) == 1
            and free_pages.dim() == 1 and free_count.numel() == 1 and lengths.is_contiguous()
            and second.is_contiguous() and free_pages.is_contiguous()
            and (lengths_out is None or lengths_out is lengths)
            and (free_count_out is None or free_count_out is free_count)
        )
    except (AttributeError, TypeError, RuntimeError):
        return False


def _check_tables(what, lengths, second, block_table, free_pages, free_count, lengths_out, free_count_out):
    _check_int32(what, lengths=lengths, block_table=block_table, free_pages=free_pages, free_count=free_count)
    if lengths.ndim != 1 or second.shape != lengths.shape:
        raise ValueError(f"{what}: lengths and the per-request tensor beside it must both be [requests]")
    _check_table(what, block_table, lengths.shape[0])
    if free_pages.ndim != 1 or free_count.numel() != 1:
        raise ValueError(f"{what}: free_pages must be [pages] and free_count hold one number")
    outs = [t for t in (lengths_out, free_count_out) if t is not None]
    for t, like, name in ((lengths_out, lengths, "lengths_out"), (free_count_out, free_count, "free_count_out")):
        if t is not None:
            _check_int32(what, **{name: t})
            if t.shape != like.shape:
                raise ValueError(f"{what}: {name} has the wrong shape")
    if not all(t.is_contiguous() for t in (lengths, second, free_pages, free_count, *outs)):
        raise ValueError(f"{what}: lengths, free_pages and free_count must be contiguous")
    _check_device(what, lengths, second, block_table, free_pages, free_count, *outs)


def reserve_pages(
    lengths: torch.Tensor,
    new_lengths: torch.Tensor,
    block_table: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    *,
    page_size: int,
    num_tokens: Optional[int] = None,
    tokens_per_request: Optional[int] = None,
    lengths_out: Optional[torch.Tensor] = None,
    free_count_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Pages, table entries and slots for the tokens that each request brings.

    All tensors int32: lengths and new_lengths [B]; block_table [B, max_pages],
    completed in place; free_pages [pages], of which the first free_count [1]
    entries are a stack of the pages that nobody owns.  Requests are served in
    order.  One whose pages would not fit its table row, or that the stack
    cannot serve after those before it, is refused: its length stays, and its
    tokens get slot -1.

    Slots are packed or padded.  num_tokens is the number of packed slots to
    write, request after request, normally the sum of new_lengths (a larger one
    leaves -1 behind them, so that a captured step can keep one size; with a
    smaller one the requests whose tokens end past it are refused).
    tokens_per_request gives every request that many, with -1 behind its last
    token: the slots of rows [B, Hkv, tokens_per_request, D].  A request that
    brings more is refused.  Returns ``(slots, starts, lengths_out,
    free_count_out)``: int64 slots; int32 starts [B + 1], where each request's
    slots begin; the new lengths and count.  lengths_out=lengths and free_count_out=free_count update in place.
    """
    what = "reserve_pages"
    index = lengths.get_device() if isinstance(lengths, torch.Tensor) else -1
    if not _tables_good(index, lengths, new_lengths, block_table, free_pages, free_count, lengths_out,
                        free_count_out) or new_lengths.dtype is not _INT32:
        _check_int32(what, new_lengths=new_lengths)
        _check_tables(what, lengths, new_lengths, block_table, free_pages, free_count, lengths_out, free_count_out)
    b = lengths.shape[0]
    if (num_tokens is None) == (tokens_per_request is None):
        raise ValueError(f"{what}: give num_tokens or tokens_per_request")
    per_request = 0
    if num_tokens is None:
        per_request = _whole(tokens_per_request)
        if per_request <= 0:
            raise ValueError(f"{what}: tokens_per_request must be positive")
        num_tokens = per_request * b
    elif _whole(num_tokens) < 0:
        raise ValueError(f"{what}: num_tokens must not be negative")
    slots = lengths.new_empty(num_tokens, dtype=_INT64)
    starts = lengths.new_empty(b + 1)
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    if free_count_out is None:
        free_count_out = torch.empty_like(free_count)
    rc = _ext.load().kf_paged_reserve(_pack_reserve(
        lengths.data_ptr(), b, block_table.data_ptr(), block_table.shape[1], block_table.stride(0),
        free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), _whole(page_size), lengths_out.data_ptr(),
        free_count_out.data_ptr(), _raw_stream(index), new_lengths.data_ptr(), slots.data_ptr(),
        num_tokens, per_request, starts.data_ptr(),
    ))
    if rc:
        _ext.check(rc, "kf_paged_reserve")
    return slots, starts, lengths_out, free_count_out


def release_pages(
    lengths: torch.Tensor,
    finished: torch.Tensor,
    block_table: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    *,
    page_size: int,
    lengths_out: Optional[torch.Tensor] = None,
    free_count_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Push the pages of finished requests (bool [B]) on the stack.

    In order of requests and positions, into free_pages in place; entries that
    are no pages of the pool are left out.  Returns ``(lengths_out,
    free_count_out)``, the finished requests' lengths being 0; their table
    rows keep old entries, which no length reaches any more.
    """
    what = "release_pages"
    if not isinstance(finished, torch.Tensor) or finished.dtype is not _BOOL:
        raise TypeError(f"{what}: finished must be a bool tensor")
    index = lengths.get_device() if isinstance(lengths, torch.Tensor) else -1
    if not _tables_good(index, lengths, finished, block_table, free_pages, free_count, lengths_out, free_count_out):
        _check_tables(what, lengths, finished, block_table, free_pages, free_count, lengths_out, free_count_out)
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    if free_count_out is None:
        free_count_out = torch.empty_like(free_count)
    rc = _ext.load().kf_paged_release(_pack_release(
        lengths.data_ptr(), lengths.shape[0], block_table.data_ptr(), block_table.shape[1], block_table.stride(0),
        free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), _whole(page_size), lengths_out.data_ptr(),
        free_count_out.data_ptr(), _raw_stream(index), finished.data_ptr(),
    ))
    if rc:
        _ext.check(rc, "kf_paged_release")
    return lengths_out, free_count_out


class PagedKVCache:
    """Pools, block table, lengths and free stack of a batch of request slots.

    ``layers`` pools share one block table, so a step reserves once and then
    appends and attends layer by layer.  Row b of the table belongs to request
    slot b; a slot of length 0 is empty.  Not thread-safe.

        cache = PagedKVCache(pages, 16, hkv, d, max_requests, max_pages, device=..., dtype=...)
        slots, starts = cache.reserve(prompt_lengths, num_tokens=n)  # prompts
        cache.append(k, v, slots)                                    # [1, Hkv, n, D]
        slots, _ = cache.reserve(active, tokens_per_request=1)       # then, token by token
        out = cache.append_and_attend(q, k, v, slots)                # [max_requests, Hq, 1, D]
        cache.release(finished)
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, max_requests: int,
                 max_pages: int, *, layers: int = 1, device: Union[torch.device, str],
                 dtype: torch.dtype) -> None:
        dims = {"num_pages": num_pages, "page_size": page_size, "kv_heads": kv_heads, "head_dim": head_dim,
                "max_requests": max_requests, "max_pages": max_pages, "layers": layers}
        for name, value in dims.items():
            if isinstance(value, bool) or not isinstance(value, int) or value <= 0:
                raise ValueError(f"{name} must be a positive integer")
        self.page_size = page_size
        self.k = torch.empty((layers, num_pages, kv_heads, page_size, head_dim), device=device, dtype=dtype)
        self.v = torch.empty_like(self.k)
        self.block_table = torch.full((max_requests, max_pages), -1, device=device, dtype=torch.int32)
        self.lengths = torch.zeros(max_requests, device=device, dtype=torch.int32)
        # the stack gives out page 0 first
        self.free_pages = torch.arange(num_pages - 1, -1, -1, device=device, dtype=torch.int32)
        self.free_count = torch.full((1,), num_pages, device=device, dtype=torch.int32)

    def reserve(self, new_lengths: torch.Tensor, *, num_tokens: Optional[int] = None,
                tokens_per_request: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Room for new_lengths (int32 [max_requests]) more tokens; advances
        ``lengths``.  Returns ``(slots, starts)`` of ``reserve_pages``, packed
        or padded as there."""
        slots, starts, _, _ = reserve_pages(
            self.lengths, new_lengths, self.block_table, self.free_pages, self.free_count,
            page_size=self.page_size, num_tokens=num_tokens, tokens_per_request=tokens_per_request,
            lengths_out=self.lengths, free_count_out=self.free_count)
        return slots, starts

    def append(self, new_k: torch.Tensor, new_v: torch.Tensor, slots: torch.Tensor, *, layer: int = 0) -> None:
        """Store K/V rows [N, Hkv, S, D] at the slots that ``reserve`` gave."""
        append_paged_kv(self.k[layer], self.v[layer], new_k, new_v, slots)

    def attend(self, q: torch.Tensor, *, layer: int = 0, scale: Optional[float] = None,
               return_lse: bool = False):
        """One query token per request slot [max_requests, Hq, 1, D] over its pages."""
        return paged_attention(q, self.k[layer], self.v[layer], self.block_table, self.lengths, scale=scale,
                               return_lse=return_lse)

    def append_and_attend(self, q: torch.Tensor, new_k: torch.Tensor, new_v: torch.Tensor, slots: torch.Tensor, *,
                          layer: int = 0, scale: Optional[float] = None, return_lse: bool = False):
        """Store the newest K/V row [max_requests, Hkv, 1, D] of every request
        and attend, in one pass.  slots come from ``reserve`` with
        tokens_per_request=1; requests without one there (no new token, or
        refused) store nothing and attend to what they have."""
        return paged_attention(q, self.k[layer], self.v[layer], self.block_table, self.lengths, scale=scale,
                               new_k=new_k, new_v=new_v, slots=slots, return_lse=return_lse)

    def release(self, finished: torch.Tensor) -> None:
        """Give up the pages of the request slots marked in finished (bool [max_requests])."""
        release_pages(self.lengths, finished, self.block_table, self.free_pages, self.free_count,
                      page_size=self.page_size, lengths_out=self.lengths, free_count_out=self.free_count)
