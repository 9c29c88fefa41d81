# SPDX-License-Identifier: Apache-2.0
"""Paged KV-cache oracle: the definitions, request by request, in 64 bits on the CPU."""
from __future__ import annotations

import math

import torch


def visible_slots(table_row, length: int, page_size: int, num_pages: int):
    """(page, row) of each position below length that the table gives a page of the pool."""
    capacity = len(table_row) * page_size
    out = []
    for p in range(max(0, min(length, capacity))):
        page = table_row[p // page_size]
        if 0 <= page < num_pages:
            out.append((page, p % page_size))
    return out


def attention(q, k_pages, v_pages, block_table, lengths, scale):
    """(O, LSE) in float64 [B, Hq, 1, D], [B, Hq, 1], and for each request the
    largest sum_i |q_i k_ji| * |scale|, the largest |v| and the number of
    visible positions, from which error bounds follow."""
    B, Hq, _, D = q.shape
    pages, Hkv, page_size, _ = k_pages.shape
    G = Hq // Hkv
    out = torch.zeros(B, Hq, 1, D, dtype=torch.float64)
    lse = torch.full((B, Hq, 1), -math.inf, dtype=torch.float64)
    sizes = []
    table, lens = block_table.cpu().tolist(), lengths.cpu().tolist()
    dev = k_pages.device
    for b in range(B):
        at = visible_slots(table[b], lens[b], page_size, pages)
        if not at:
            sizes.append((0.0, 0.0, 0))
            continue
        page = torch.tensor([x[0] for x in at], device=dev)
        row = torch.tensor([x[1] for x in at], device=dev)
        k = k_pages[page, :, row].cpu().double().permute(1, 0, 2)  # [Hkv, n, D]
        v = v_pages[page, :, row].cpu().double().permute(1, 0, 2)
        qb = q[b, :, 0].cpu().double().view(Hkv, G, D)
        x = torch.matmul(qb, k.transpose(1, 2)) * scale
        top = x.max(-1, keepdim=True).values
        w = torch.exp(x - top)
        total = w.sum(-1, keepdim=True)
        out[b, :, 0] = (torch.matmul(w, v) / total).reshape(Hq, D)
        lse[b, :, 0] = (torch.log(total) + top).reshape(Hq)
        sizes.append(((torch.matmul(qb.abs(), k.abs().transpose(1, 2)).max() * abs(scale)).item(),
                      v.abs().max().item(), len(at)))
    return out, lse, sizes


def reserve(lengths, added, table, free_pages, free_count, page_size, num_tokens=None, per_request=None):
    """Lists in, lists out: (slots, starts, lengths, count, table); the stack is free_pages[:free_count]."""
    num_pages = len(free_pages)
    table = [list(r) for r in table]
    count = max(0, min(free_count, num_pages))
    claimed = 0  # by the requests so far, granted or not
    taken = 0
    slots, starts, new_lengths = [], [0], []
    for b, (n, m) in enumerate(zip(lengths, added)):
        n, m = max(n, 0), max(m, 0)
        before, after = -(-n // page_size), -(-(n + m) // page_size)
        need = after - before
        fits = after <= len(table[b]) and n + m < 2**31 and (per_request is None or m <= per_request)
        if fits:
            claimed += need
        slotted = per_request is not None or m == 0 or len(slots) + m <= num_tokens
        granted = fits and slotted and (need == 0 or claimed <= count)
        if granted:
            for j in range(need):
                table[b][before + j] = free_pages[count - 1 - taken - j]
            taken += need
        mine = []
        for p in range(n, n + m):
            page = table[b][p // page_size] if granted else -1
            mine.append(page * page_size + p % page_size if 0 <= page < num_pages else -1)
        if per_request is not None:
            mine = (mine + [-1] * per_request)[:per_request]
        slots += mine
        starts.append(len(slots))
        new_lengths.append(n + m if granted else n)
    if per_request is None:
        slots = (slots + [-1] * num_tokens)[:num_tokens]
    return slots, starts, new_lengths, count - taken, table


def release(lengths, finished, table, free_pages, free_count, page_size):
    """Lists in, lists out: (lengths, count, free_pages)."""
    num_pages = len(free_pages)
    free = list(free_pages)
    count = max(0, min(free_count, num_pages))
    out = []
    for b, (n, gone) in enumerate(zip(lengths, finished)):
        n = max(n, 0)
        if gone:
            for page in table[b][: min(-(-n // page_size), len(table[b]))]:
                if 0 <= page < num_pages and count < num_pages:
                    free[count] = page
                    count += 1
        out.append(0 if gone else n)
    return out, count, free
