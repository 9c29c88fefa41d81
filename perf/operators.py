# SPDX-License-Identifier: Apache-2.0
"""The paged KV-cache operators: what each computes, at sizes that stand for its use.

A server keeps the keys and values of all its requests in one pool of pages,
``k_pages`` and ``v_pages`` [pages, Hkv, page_size, D].  A block table
[requests, max_pages] names the pages of each request in order, and a stack of
free pages holds the rest.  One serving step is

* ``reserve``: from the requests' lengths and how many tokens each brings,
  take the pages that they need from the stack, enter them in the block table
  and give each new token its slot (page * page_size + offset in the page);
* ``append``: copy the new tokens' K/V rows to their slots (a prompt);
* ``attend``: one query token of each request over the request's pages;
* ``step``: the same with the newest token's K/V row written to its slot on
  the way (generation);
* ``release``: push the pages of finished requests back on the stack.

``run`` computes them in elementary torch operations, in 32 bits and rounded
once, or with ``own`` through the package's entry points.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the shortest call: one request that has just begun, in a small grouped-query model; latency alone
        dict(name="attend_one_short", op="attend", B=1, Hq=8, Hkv=2, D=64, dtype="f16", page=16, low=33, high=33, lse=False),
        # two long documents, few heads: the split over the length carries it
        dict(name="attend_two_long", op="attend", B=2, Hq=8, Hkv=2, D=64, dtype="f16", page=64, low=131072, high=131072, lse=True),
        # a full server: 64 requests of mixed ages, 32 query and 8 KV heads
        dict(name="attend_batch_ragged", op="attend", B=64, Hq=32, Hkv=8, D=128, dtype="bf16", page=16, low=128, high=8192, lse=False),
        # odd everything: a head dim off the powers of two, pages that end inside a tile, an empty request
        dict(name="attend_odd", op="attend", B=7, Hq=16, Hkv=4, D=72, dtype="bf16", page=24, low=0, high=5003, lse=True),
        # generation with the append fused in, 8 requests at about 4096 tokens
        dict(name="step_batch8", op="step", B=8, Hq=32, Hkv=8, D=128, dtype="bf16", page=16, low=4096, high=4352, lse=False),
        # many query heads on one KV head, short contexts
        dict(name="step_shared_head", op="step", B=32, Hq=32, Hkv=1, D=96, dtype="f16", page=32, low=1, high=2047, lse=False),
        # one token of each of 256 requests into the pool
        dict(name="append_tokens", op="append", T=256, Hkv=8, D=128, dtype="bf16", page=16),
        # prompts, 16384 tokens in all
        dict(name="append_prompts", op="append", T=16384, Hkv=8, D=128, dtype="bf16", page=16),
        # the tables of a generation step: one token for each of 256 requests
        dict(name="reserve_tokens", op="reserve", B=256, page=16, low=100, high=8000, new_low=1, new_high=1),
        # the tables of 48 new prompts, 100 to 5000 tokens each
        dict(name="reserve_prompts", op="reserve", B=48, page=16, low=0, high=0, new_low=100, new_high=5000),
        # a few short requests end
        dict(name="release_few", op="release", B=16, page=16, low=10, high=900, every=3),
        # a quarter of a full server ends
        dict(name="release_many", op="release", B=256, page=16, low=100, high=8000, every=4),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "step", "step", "append", "reserve", "release"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    D = rng.choice([16, 40, 64, 64, 72, 96, 104, 128, 128, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8, 16])
    dtype = rng.choice(["f16", "bf16"])
    if op == "append":
        T = _log(rng, 1, max(1, min(65536, 16384 * 8 * 128 // (Hkv * D))))
        return dict(op=op, T=T, Hkv=Hkv, D=D, dtype=dtype, page=page)
    if op == "reserve":
        B = _log(rng, 1, 512)
        new_high = _log(rng, 1, max(1, 120000 // B))
        high = rng.choice([0, _log(rng, 1, 8000)])
        return dict(op=op, B=B, page=page, low=high // 8, high=high, new_low=rng.randint(0, new_high), new_high=new_high)
    if op == "release":
        high = _log(rng, 1, 8000)
        return dict(op=op, B=_log(rng, 1, 256), page=page, low=rng.randint(0, high), high=high, every=rng.randint(1, 6))
    G = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 12, 16, 32])
    while Hkv * G > 64:
        G = max(1, G // 2)
    B = _log(rng, 1, 256)
    most = min(131072, 64 * 8192 * 8 * 128 // (B * Hkv * max(D, 64)), 64 * 8192 * 32 * 128 // (B * Hkv * G * max(D, 64)))
    high = _log(rng, 1, max(1, most))
    low = rng.choice([0, 1, high // 2, high])
    return dict(op=op, B=B, Hq=Hkv * G, Hkv=Hkv, D=D, dtype=dtype, page=page, low=min(low, high) if op == "attend" else max(1, min(low, high)),
                high=high, lse=rng.choice([False, True]) if op == "attend" else False)


def _spread(low, high, n):
    """n whole numbers from low to high in even steps: their sum is the case's own, their order the seed's."""
    return [high] if n == 1 else [low + (high - low) * i // (n - 1) for i in range(n)]


def _pages(n, page):
    return -(-n // page)


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    op, page = case["op"], case["page"]

    def order(n):
        return torch.randperm(n, generator=g, device=dev)

    def normal(*shape, scale=1.0):
        x = torch.randn(*shape, generator=g, device=dev, dtype=DTYPES[case["dtype"]])
        return x if scale == 1.0 else x * scale

    s = {"case": case}
    if op == "append":
        T, Hkv, D = case["T"], case["Hkv"], case["D"]
        n = 2 * _pages(T, page) + 3
        s["k_pages"], s["v_pages"] = normal(n, Hkv, page, D), normal(n, Hkv, page, D)
        # prompts fill whole pages one after another, single tokens fall anywhere
        if T >= 1024:
            slots = (order(n)[: _pages(T, page)][:, None] * page + torch.arange(page, device=dev)).reshape(-1)[:T]
        else:
            slots = order(n * page)[:T]
        s["slots"] = slots.to(torch.int64).contiguous()
        # as the projection gives them: tokens first, heads and columns inside
        s["new_k"], s["new_v"] = normal(1, T, Hkv, D).transpose(1, 2), normal(1, T, Hkv, D).transpose(1, 2)
        return s

    B = case["B"]
    lens = torch.tensor(_spread(case["low"], case["high"], B), device=dev)[order(B)].to(torch.int32)
    held = (lens + page - 1) // page
    if op in ("reserve", "release"):
        if op == "reserve":
            new = torch.tensor(_spread(case["new_low"], case["new_high"], B), device=dev)[order(B)].to(torch.int32)
            s["new"] = new
            s["T"] = sum(_spread(case["new_low"], case["new_high"], B))
            width = _pages(case["high"] + case["new_high"], page) + 1
        else:
            s["finished"] = torch.arange(B, device=dev)[order(B)] % case["every"] == 0
            width = _pages(case["high"], page) + 1
        n = B * width + 7
        pages = order(n).to(torch.int32)
        cols = torch.arange(width, device=dev)
        s["block_table"] = torch.where(cols < held[:, None], pages[: B * width].view(B, width), -1).to(torch.int32).contiguous()
        used = int(held.sum())
        left = torch.cat((pages[: B * width].view(B, width)[cols >= held[:, None]], pages[B * width:]))
        s["free_pages"] = torch.cat((left, torch.full((n - left.numel(),), -1, dtype=torch.int32, device=dev))).contiguous()
        s["free_count"] = torch.tensor([n - used], dtype=torch.int32, device=dev)
        s["lengths"] = lens
        return s

    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    width = max(1, _pages(case["high"], page))
    n = sum(_pages(x, page) for x in _spread(case["low"], case["high"], B)) + 5
    pages = order(n).to(torch.int32)
    first = torch.cumsum(held, 0) - held
    cols = torch.arange(width, device=dev)
    s["block_table"] = torch.where(cols < held[:, None], pages[(first[:, None] + cols).clamp(max=n - 1)], -1).to(torch.int32).contiguous()
    s["lengths"] = lens
    s["k_pages"], s["v_pages"] = normal(n, Hkv, page, D), normal(n, Hkv, page, D)
    s["q"] = normal(B, Hq, 1, D, scale=1.5)
    s["scale"] = D ** -0.5
    if op == "step":
        s["new_k"], s["new_v"] = normal(B, Hkv, 1, D), normal(B, Hkv, 1, D)
        last = lens.long() - 1
        s["slots"] = s["block_table"].gather(1, (last // page)[:, None])[:, 0].long() * page + last % page
    return s


# ---------------------------------------------------------------- plain forms

def _attend(q, k_pages, v_pages, table, lengths, scale):
    B, Hq, _, D = q.shape
    Hkv, page = k_pages.shape[1], k_pages.shape[2]
    at = table.clamp(min=0).long()
    keys = at.shape[1] * page

    def rows(pages):
        return pages[at].transpose(1, 2).reshape(B, Hkv, keys, D).float()

    seen = (torch.arange(keys, device=q.device) < lengths[:, None])[:, None, None, :]
    scores = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, D), rows(k_pages).transpose(-1, -2)) * scale
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, rows(v_pages)) / torch.where(total == 0, 1.0, total)
    lse = torch.log(total) + top
    return out.view(B, Hq, 1, D).to(q.dtype), lse.view(B, Hq, 1)


def _append(k_pages, v_pages, new_k, new_v, slots):
    Hkv, page, D = k_pages.shape[1:]
    at, inside = slots // page, slots % page
    k_pages[at, :, inside] = new_k.transpose(1, 2).reshape(-1, Hkv, D)
    v_pages[at, :, inside] = new_v.transpose(1, 2).reshape(-1, Hkv, D)


def _reserve(lengths, new, table, free, count, page, T):
    """A request whose pages do not fit the table, or the stack after those before it, brings nothing."""
    B, width = table.shape
    before, after = (lengths + page - 1) // page, (lengths + new + page - 1) // page
    fits = after <= width
    need = torch.where(fits, after - before, 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= count))
    first = upto - need
    ends = torch.cumsum(new, 0)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends)).to(torch.int32)
    cols = torch.arange(width, device=table.device)
    fresh = granted[:, None] & (cols >= before[:, None]) & (cols < after[:, None])
    source = count - 1 - (first[:, None] + cols - before[:, None])
    table.copy_(torch.where(fresh, free[source.clamp(0, free.numel() - 1)], table))
    token = torch.arange(T, device=table.device)
    b = torch.searchsorted(ends, token, right=True).clamp(max=B - 1)
    position = lengths[b] + token - starts[b]
    slots = table[b, (position // page).clamp(max=width - 1)].long() * page + position % page
    slots = torch.where(granted[b], slots, -1)
    taken = torch.where(granted, need, 0).sum()
    return slots, starts, (lengths + torch.where(granted, new, 0)).to(torch.int32), (count - taken).to(torch.int32)


def _release(lengths, finished, table, free, count, page):
    B, width = table.shape
    N = free.numel()
    cols = torch.arange(width, device=table.device)
    gone = finished[:, None] & (cols < ((lengths + page - 1) // page)[:, None]) & (table >= 0) & (table < N)
    at = torch.cumsum(gone.view(-1), 0) - 1 + count
    at = torch.where(gone.view(-1) & (at < N), at, N)
    free.copy_(torch.cat((free, free[:1])).scatter(0, at, table.view(-1))[:N])
    return torch.where(finished, 0, lengths).to(torch.int32), (count + gone.sum()).clamp(max=N).to(torch.int32)


def run(state):
    s, case = state, state["case"]
    op, page = case["op"], case["page"]
    if own:
        from kotflash_b200 import paged
    if op == "attend":
        if own:
            r = paged.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], scale=s["scale"], return_lse=case["lse"])
            return r
        out, lse = _attend(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], s["scale"])
        return (out, lse) if case["lse"] else out
    if op == "step":
        if own:
            out = paged.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], scale=s["scale"], new_k=s["new_k"], new_v=s["new_v"],
                                       slots=s["slots"])
        else:
            _append(s["k_pages"], s["v_pages"], s["new_k"], s["new_v"], s["slots"])
            out, _ = _attend(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], s["scale"])
        return out, s["k_pages"], s["v_pages"]
    if op == "append":
        if own:
            paged.append_paged_kv(s["k_pages"], s["v_pages"], s["new_k"], s["new_v"], s["slots"])
        else:
            _append(s["k_pages"], s["v_pages"], s["new_k"], s["new_v"], s["slots"])
        return s["k_pages"], s["v_pages"]
    if op == "reserve":
        if own:
            slots, starts, lengths, count = paged.reserve_pages(s["lengths"], s["new"], s["block_table"], s["free_pages"], s["free_count"], page_size=page,
                                                                num_tokens=s["T"])
        else:
            slots, starts, lengths, count = _reserve(s["lengths"], s["new"], s["block_table"], s["free_pages"], s["free_count"], page, s["T"])
        return slots, starts, lengths, count, s["block_table"]
    if own:
        lengths, count = paged.release_pages(s["lengths"], s["finished"], s["block_table"], s["free_pages"], s["free_count"], page_size=page)
    else:
        lengths, count = _release(s["lengths"], s["finished"], s["block_table"], s["free_pages"], s["free_count"], page)
    return lengths, count, s["free_pages"]


def work(case):
    op, page = case["op"], case["page"]
    if op == "append":
        row = case["Hkv"] * case["D"] * 2
        return {"bytes": case["T"] * (4 * row + 8), "flops": 0}
    B = case["B"]
    lens = _spread(case["low"], case["high"], B)
    if op == "reserve":
        new = _spread(case["new_low"], case["new_high"], B)
        fresh = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(lens, new))
        return {"bytes": 8 * sum(new) + 8 * fresh + 16 * B + 12, "flops": 0}
    if op == "release":
        gone = sum(_pages(x, page) for x in lens) / max(1, case["every"])
        return {"bytes": 8 * gone + 9 * B + 8, "flops": 0}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    moved = sum(lens) * Hkv * D * 4 + 2 * B * Hq * D * 2 + 4 * B + 4 * sum(_pages(x, page) for x in lens)
    if case["lse"]:
        moved += 4 * B * Hq
    if op == "step":
        moved += 4 * B * Hkv * D * 2 - 4 * B * Hkv * D  # the new rows come from the caller instead of the pool, and go there
    return {"bytes": moved, "flops": 4 * sum(lens) * Hq * D}


def exact(case, seed):
    """The definition, request by request, in 64 bits."""
    if case["op"] in ("reserve", "release"):
        return None
    s = prepare(case, seed)
    page = case["page"]
    k, v = s["k_pages"], s["v_pages"]
    if case["op"] == "append":
        new_k, new_v = s["new_k"][0], s["new_v"][0]
        flat_k, flat_v = (x.permute(0, 2, 1, 3).reshape(-1, case["Hkv"], case["D"]) for x in (k.double(), v.double()))
        flat_k[s["slots"]] = new_k.permute(1, 0, 2).double()
        flat_v[s["slots"]] = new_v.permute(1, 0, 2).double()
        return tuple(x.view(-1, page, case["Hkv"], case["D"]).permute(0, 2, 1, 3) for x in (flat_k, flat_v))
    lens, table = s["lengths"].tolist(), s["block_table"].long()
    if case["op"] == "step":
        for b, n in enumerate(lens):
            at, inside = int(table[b, (n - 1) // page]), (n - 1) % page
            k[at, :, inside], v[at, :, inside] = s["new_k"][b, :, 0], s["new_v"][b, :, 0]
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    out = torch.zeros(B, Hq, 1, D, dtype=torch.float64, device=k.device)
    lse = torch.full((B, Hq, 1), -math.inf, dtype=torch.float64, device=k.device)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        mine = table[b, : _pages(n, page)]
        kb, vb = (x[mine].permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n].double() for x in (k, v))
        x = torch.einsum("hgd,hnd->hgn", s["q"][b, :, 0].double().view(Hkv, -1, D), kb) * s["scale"]
        lse[b, :, 0] = torch.logsumexp(x, -1).view(-1)
        out[b, :, 0] = torch.einsum("hgn,hnd->hgd", torch.softmax(x, -1), vb).reshape(Hq, D)
    if case["op"] == "step":
        return out, k.double(), v.double()
    return (out, lse) if case["lse"] else out
