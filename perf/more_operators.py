# SPDX-License-Identifier: Apache-2.0
"""Rotary positions and the 8-bit paged KV cache: what each operator computes, at sizes that stand for its use.

A step of a model rotates its queries and keys by their positions, stores the
keys and values in the cache and attends to it:

* ``rotate``: columns of q and k as pairs, each turned by position * frequency
  (halves of the rotated columns or neighbours as pairs; the columns behind
  them pass); ``rotate_train`` with the gradients;
* ``store``: K/V rows to their slots of a pool of pages, in 8 bits with a
  power of two as the scale of each block of tokens and head;
* ``load``: rows of given slots back in 16 bits;
* ``attend``: one query token of each request over the request's pages;
* ``step``: the same with the newest token's K/V row stored on the way.

A block's scale is the smallest power of two that holds its rows: 448 times it
in e4m3, 127 steps of it (after rounding) in int8, within 2^-60 and 2^60; a
block with an infinity, a NaN or more than that has the scale NaN.  Rows that
join a block that has rows already may raise its scale; those rows are then
rounded again.  Writing a block's first row begins it anew.

``run`` computes them in elementary torch operations, in 32 bits (angles in
64) and rounded once, or with ``own`` through the package's entry points.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def listed():
    return [
        # the queries and keys of a generation step: 64 requests far into long contexts
        dict(name="rotate_step", op="rotate", B=64, S=1, Hq=32, Hkv=8, D=128, R=128, dtype="bf16", pairs="halves", base=500000.0, stretch=8.0, far=131072),
        # the prefill of the attention benchmark: 4 x 4096 tokens, 32 query and 8 KV heads
        dict(name="rotate_prompts", op="rotate", B=4, S=4096, Hq=32, Hkv=8, D=128, R=128, dtype="bf16", pairs="halves", base=10000.0, stretch=1.0, far=4096),
        # a training step with its gradients, odd length, part of the head, neighbours as pairs
        dict(name="rotate_train", op="rotate_train", B=1, S=5003, Hq=16, Hkv=4, D=96, R=64, dtype="f16", pairs="neighbours", base=10000.0, stretch=1.0, far=5003),
        # prompts, 16384 tokens in all, a scale for each row
        dict(name="store_prompts", op="store", T=16384, Hkv=8, D=128, dtype="bf16", held="e4m3", page=16, block=1, runs=8),
        # prompts that go on where earlier ones ended inside a block of 16 tokens with one scale
        dict(name="store_blocks", op="store", T=4096, Hkv=8, D=128, dtype="bf16", held="int8", page=32, block=16, runs=11),
        # a long prefix back in 16 bits, for the next part of its prompt
        dict(name="load_prefix", op="load", T=16384, Hkv=8, D=128, dtype="bf16", held="e4m3", page=16, block=1),
        # a short one of an odd length, a head dim off the powers of two
        dict(name="load_odd", op="load", T=1003, Hkv=4, D=72, dtype="f16", held="int8", page=24, block=8),
        # the shortest call: one request that has just begun; latency alone
        dict(name="attend_one_short", op="attend", B=1, Hq=8, Hkv=2, D=64, dtype="f16", held="e4m3", page=16, block=1, low=33, high=33, lse=False),
        # two long documents, few heads: the split over the length carries it
        dict(name="attend_two_long", op="attend", B=2, Hq=8, Hkv=2, D=64, dtype="f16", held="int8", page=64, block=1, low=131072, high=131072, lse=True),
        # a full server: 64 requests of mixed ages, 32 query and 8 KV heads
        dict(name="attend_batch_ragged", op="attend", B=64, Hq=32, Hkv=8, D=128, dtype="bf16", held="e4m3", page=16, block=1, low=128, high=8192, lse=False),
        # odd everything: head dim, pages that end inside a tile, an empty request, blocks of 8 tokens
        dict(name="attend_odd", op="attend", B=7, Hq=16, Hkv=4, D=72, dtype="bf16", held="int8", page=24, block=8, low=0, high=5003, lse=True),
        # generation with the newest row stored on the way, 8 requests at about 4096 tokens
        dict(name="step_batch8", op="step", B=8, Hq=32, Hkv=8, D=128, dtype="bf16", held="e4m3", page=16, block=1, low=4096, high=4352, lse=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "rotate_train", "store", "store", "load", "attend", "attend", "attend", "step", "step"])
    dtype = rng.choice(["f16", "bf16"])
    D = rng.choice([16, 40, 64, 64, 72, 96, 104, 128, 128, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8, 16])
    G = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 12, 16, 32])
    while Hkv * G > 64:
        G = max(1, G // 2)
    if op.startswith("rotate"):
        most = 4 * 4096 * 40 * 128 // (Hkv * (G + 1) * D) // (2 if op == "rotate_train" else 1)
        T = _log(rng, 1, max(1, min(65536, most)))
        B = rng.choice([1, 1, 2, 3, 8, T])
        B = min(B, T)
        S = max(1, T // B)
        stretch = rng.choice([1.0, 1.0, 4.0, 8.0])
        return dict(op=op, B=B, S=S, Hq=Hkv * G, Hkv=Hkv, D=D, R=rng.choice([D, D, D // 2 // 2 * 2, D // 4 // 2 * 2]), dtype=dtype,
                    pairs=rng.choice(["halves", "halves", "neighbours"]), base=rng.choice([10000.0, 500000.0, 1000000.0]), stretch=stretch,
                    far=max(S, rng.choice([S, 4096, 32768, 131072])))
    held = rng.choice(["e4m3", "e4m3", "int8"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    block = rng.choice([1, 1, 1, 8, 8 if page % 16 else 16])
    if op in ("store", "load"):
        T = _log(rng, 1, max(1, min(65536, 16384 * 8 * 128 // (Hkv * max(D, 64)) // (4 if block > 1 and op == "store" else 1))))
        c = dict(op=op, T=T, Hkv=Hkv, D=D, dtype=dtype, held=held, page=page, block=block)
        if op == "store":
            c["runs"] = rng.choice([1, min(T, 8), T if T <= 512 else 16])
        return c
    B = _log(rng, 1, 256)
    most = min(131072, 64 * 4096 * 8 * 128 // (B * Hkv * max(D, 64)), 64 * 4096 * 32 * 128 // (B * Hkv * G * max(D, 64)))
    high = _log(rng, 1, max(1, most))
    low = rng.choice([0, 1, high // 2, high])
    return dict(op=op, B=B, Hq=Hkv * G, Hkv=Hkv, D=D, dtype=dtype, held=held, page=page, block=block, high=high,
                low=min(low, high) if op == "attend" else max(1, min(low, high)), lse=rng.choice([False, True]) if op == "attend" else False)


def _spread(low, high, n):
    """n whole numbers from low to high in even steps: their sum is the case's own, their order the seed's."""
    return [high] if n == 1 else [low + (high - low) * i // (n - 1) for i in range(n)]


def _pages(n, page):
    return -(-n // page)


def _frequencies(case, dev):
    """Radians per position of each pair: base^(-2i / R), the slow ones (under one turn in 8192 positions) stretched, those between blended."""
    f = case["base"] ** (-torch.arange(0, case["R"], 2, dtype=torch.float64, device=dev) / case["R"])
    if case["stretch"] != 1.0:
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        f = f * keep + f / case["stretch"] * (1 - keep)
    return f


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    op, D, Hkv = case["op"], case["D"], case["Hkv"]

    def order(n):
        return torch.randperm(n, generator=g, device=dev)

    def normal(*shape, scale=1.0):
        x = torch.randn(*shape, generator=g, device=dev, dtype=DTYPES[case["dtype"]])
        return x if scale == 1.0 else x * scale

    s = {"case": case}
    if op.startswith("rotate"):
        B, S, Hq = case["B"], case["S"], case["Hq"]
        # as one product gives them: tokens first, the heads of q, k and v side by side
        rows = normal(B, S, Hq + 2 * Hkv, D).transpose(1, 2)
        s["q"], s["k"], _ = rows.split([Hq, Hkv, Hkv], 1)
        first = torch.randint(0, case["far"] - S + 1, (B, 1), generator=g, device=dev)
        s["positions"] = (first + torch.arange(S, device=dev)).to(torch.int32)
        s["frequencies"] = _frequencies(case, dev)
        s["magnitude"] = 1.0 if case["stretch"] == 1.0 else 0.1 * math.log(case["stretch"]) + 1.0
        if op == "rotate_train":
            s["q"], s["k"] = (x.detach().requires_grad_(True) for x in (s["q"], s["k"]))
            # attention gives its gradients heads first
            s["dq"], s["dk"] = normal(B, Hq, S, D), normal(B, Hkv, S, D)
        return s

    page, block = case["page"], case["block"]

    def pool(n):
        """Codes as rows of normal values have them, scales around 2^-7; rows start on 16 bytes."""
        x = torch.empty(n, Hkv, page, -(-D // 16) * 16, device=dev, dtype=DTYPES[case["held"]])[..., :D]
        for part in x.split(max(1, (1 << 26) // (Hkv * page * D))):
            y = torch.randn(part.shape, generator=g, device=dev, dtype=torch.float16)
            part.copy_((y * 100).clamp(-448, 448) if case["held"] == "e4m3" else (y * 35).round().clamp(-127, 127))
        e = torch.randint(127 - 8, 127 - 5, (n, Hkv, page // block), generator=g, device=dev, dtype=torch.uint8)
        return x, e.view(torch.float8_e8m0fnu)

    if op in ("store", "load"):
        T = case["T"]
        n = 2 * _pages(T, page) + 2 * case.get("runs", 1) + 3
        s["k_pages"], s["k_scales"] = pool(n)
        s["v_pages"], s["v_scales"] = pool(n)
        # runs of tokens, each behind the rows of an earlier one in its first page, pages anywhere
        runs = case.get("runs", 1)
        sizes = [T // runs + (i < T % runs) for i in range(runs)]
        before = torch.randint(0, page, (runs,), generator=torch.Generator().manual_seed(seed)).tolist()
        pages, at, slots = order(n), 0, []
        for size, b in zip(sizes, before):
            held = pages[at: at + _pages(b + size, page)]
            at += held.numel()
            slots.append((held[:, None] * page + torch.arange(page, device=dev)).reshape(-1)[b: b + size])
        s["slots"] = torch.cat(slots).to(torch.int64).contiguous()
        if op == "store":
            s["new_k"], s["new_v"] = normal(1, T, Hkv, D).transpose(1, 2), normal(1, T, Hkv, D).transpose(1, 2)
        return s

    B, Hq = case["B"], case["Hq"]
    lens = torch.tensor(_spread(case["low"], case["high"], B), device=dev)[order(B)].to(torch.int32)
    held = (lens + page - 1) // page
    width = max(1, _pages(case["high"], page))
    n = sum(_pages(x, page) for x in _spread(case["low"], case["high"], B)) + 5
    pages = order(n).to(torch.int32)
    first = torch.cumsum(held, 0) - held
    cols = torch.arange(width, device=dev)
    s["block_table"] = torch.where(cols < held[:, None], pages[(first[:, None] + cols).clamp(max=n - 1)], -1).to(torch.int32).contiguous()
    s["lengths"] = lens
    s["k_pages"], s["k_scales"] = pool(n)
    s["v_pages"], s["v_scales"] = pool(n)
    s["q"] = normal(B, Hq, 1, D, scale=1.5)
    s["scale"] = D ** -0.5
    if op == "step":
        s["new_k"], s["new_v"] = normal(B, Hkv, 1, D), normal(B, Hkv, 1, D)
        last = lens.long() - 1
        s["slots"] = s["block_table"].gather(1, (last // page)[:, None])[:, 0].long() * page + last % page
    return s


# ---------------------------------------------------------------- plain forms

def _turn(x, cos, sin, pairs, R):
    """Each pair (a, b) of the first R columns becomes (a cos - b sin, b cos + a sin)."""
    y = x.float()
    if pairs == "halves":
        a, b = y[..., : R // 2], y[..., R // 2: R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, y[..., R:]), -1).to(x.dtype)


def _angles(positions, frequencies, magnitude):
    """cos and sin [B, 1, S, R / 2], the angles in 64 bits."""
    at = (positions.double()[..., None] * frequencies)[:, None]
    return (torch.cos(at) * magnitude).float(), (torch.sin(at) * magnitude).float()


def _exponent(top, held):
    """The scale's exponent for rows whose largest magnitude is `top`, NaN where there is none."""
    m, e = torch.frexp(top)
    e = e - 9 + (m > 0.875).int() if held == "e4m3" else e - 7 + (m >= 255 / 256).int()
    e = torch.where(top == 0, -60, e).clamp(min=-60)
    return torch.where(torch.isfinite(top) & (e <= 60), e.float(), math.nan)


def _codes(x, scale, dtype):
    y = torch.nan_to_num(x / scale, nan=0.0, posinf=0.0, neginf=0.0)
    return y.round().clamp(-127, 127).to(dtype) if dtype == torch.int8 else y.to(dtype)


def _bytes(exponent):
    return torch.where(torch.isnan(exponent), 255, exponent + 127).to(torch.uint8)


def _store(pages, scales, new, slots, held):
    """Rows [1 or N, Hkv, S, D] to their slots."""
    n, Hkv, page, D = pages.shape
    block = page // scales.shape[2]
    rows = new.transpose(1, 2).reshape(-1, Hkv, D).float()
    at, inside = slots // page, slots % page
    top = torch.nan_to_num(rows.abs(), nan=math.inf).amax(-1)  # [T, Hkv]
    raw = scales.view(torch.uint8)
    if block == 1:
        e = _exponent(top, held)
        raw[at, :, inside] = _bytes(e)
        # an index_put of 8-bit floats goes by their bytes
        pages.view(torch.uint8)[at, :, inside] = _codes(rows, torch.exp2(e)[..., None], pages.dtype).view(torch.uint8)
        return
    # per block of the pool: the largest new magnitude and the first row written
    count = n * page // block
    b = slots // block
    tops = torch.zeros(count, Hkv, device=rows.device).scatter_reduce(0, b[:, None].expand(-1, Hkv), top, "amax")
    first = torch.full((count,), block, device=rows.device).scatter_reduce(0, b, slots % block, "amin")
    e = _exponent(tops, held).view(n, page // block, Hkv).transpose(1, 2)
    first = first.view(n, 1, page // block)
    was = torch.where(raw == 255, math.nan, raw.float() - 127)
    now = torch.where(first == 0, e, torch.where(first == block, was, torch.where(torch.isnan(e) | torch.isnan(was), math.nan, torch.maximum(e, was))))
    # the rows before the first written one keep their values as far as the new scale holds them
    shift = torch.exp2(was - now).repeat_interleave(block, 2)[..., None]
    kept = (torch.arange(page, device=rows.device) % block)[None, None, :, None] < first.repeat_interleave(block, 2)[..., None]
    moved = kept & (shift != 1) & (first < block).repeat_interleave(block, 2)[..., None]
    pages.copy_(torch.where(moved, _codes(pages.float() * shift, torch.ones_like(shift), pages.dtype).float(), pages.float()).to(pages.dtype))
    raw.copy_(_bytes(now))
    scale = torch.exp2(now)[at, :, inside // block][..., None]
    pages.view(torch.uint8)[at, :, inside] = _codes(rows, scale, pages.dtype).view(torch.uint8)


def _values(codes, raw):
    """What codes [..., rows, D] with the scales' bytes [..., rows / block] stand for."""
    scale = torch.where(raw == 255, math.nan, torch.exp2(raw.float() - 127))
    return codes.float() * scale.repeat_interleave(codes.shape[-2] // raw.shape[-1], -1)[..., None]


def _load(pages, scales, slots, dtype):
    Hkv, page = pages.shape[1:3]
    block = page // scales.shape[2]
    at, inside = slots // page, slots % page
    raw = scales.view(torch.uint8)[at, :, inside // block]
    scale = torch.where(raw == 255, math.nan, torch.exp2(raw.float() - 127))
    rows = pages.view(torch.uint8)[at, :, inside].view(pages.dtype).float() * scale[..., None]
    return rows.transpose(0, 1)[None].to(dtype)


def _attend(q, k_pages, v_pages, k_scales, v_scales, table, lengths, scale):
    B, Hq, _, D = q.shape
    Hkv, page = k_pages.shape[1], k_pages.shape[2]
    at = table.clamp(min=0).long()
    keys = at.shape[1] * page

    def rows(pages, scales):
        x = _values(pages.view(torch.uint8)[at].view(pages.dtype), scales.view(torch.uint8)[at])
        return x.transpose(1, 2).reshape(B, Hkv, keys, D)

    seen = (torch.arange(keys, device=q.device) < lengths[:, None])[:, None, None, :]
    scores = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, D), rows(k_pages, k_scales).transpose(-1, -2)) * scale
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, torch.where(seen.transpose(-1, -2), rows(v_pages, v_scales), 0.0)) / torch.where(total == 0, 1.0, total)
    lse = torch.log(total) + top
    return out.view(B, Hq, 1, D).to(q.dtype), lse.view(B, Hq, 1)


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from kotflash_b200 import paged8, rotary
    if op.startswith("rotate"):
        neighbours = case["pairs"] == "neighbours"
        if own:
            out = rotary.apply_rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=neighbours, magnitude=s["magnitude"])
            if op == "rotate":
                return out
            return (*out, *torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"])))
        cos, sin = _angles(s["positions"], s["frequencies"], s["magnitude"])
        out = tuple(_turn(x.detach(), cos, sin, case["pairs"], case["R"]) for x in (s["q"], s["k"]))
        if op == "rotate":
            return out
        # the gradient of a rotation is the rotation back
        return (*out, *(_turn(x, cos, -sin, case["pairs"], case["R"]) for x in (s["dq"], s["dk"])))
    cache = tuple(s[x] for x in ("k_pages", "v_pages", "k_scales", "v_scales"))
    if op == "store":
        if own:
            paged8.append_paged_kv8(*cache, s["new_k"], s["new_v"], s["slots"])
        else:
            _store(s["k_pages"], s["k_scales"], s["new_k"], s["slots"], case["held"])
            _store(s["v_pages"], s["v_scales"], s["new_v"], s["slots"], case["held"])
        return cache
    if op == "load":
        dtype = DTYPES[case["dtype"]]
        if own:
            return paged8.read_paged_kv8(*cache, s["slots"], dtype=dtype)
        return _load(s["k_pages"], s["k_scales"], s["slots"], dtype), _load(s["v_pages"], s["v_scales"], s["slots"], dtype)
    if op == "attend":
        if own:
            return paged8.paged_attention8(s["q"], *cache, s["block_table"], s["lengths"], scale=s["scale"], return_lse=case["lse"])
        out, lse = _attend(s["q"], *cache, s["block_table"], s["lengths"], s["scale"])
        return (out, lse) if case["lse"] else out
    if own:
        out = paged8.paged_attention8(s["q"], *cache, s["block_table"], s["lengths"], scale=s["scale"], new_k=s["new_k"], new_v=s["new_v"], slots=s["slots"])
    else:
        _store(s["k_pages"], s["k_scales"], s["new_k"], s["slots"], case["held"])
        _store(s["v_pages"], s["v_scales"], s["new_v"], s["slots"], case["held"])
        out, _ = _attend(s["q"], *cache, s["block_table"], s["lengths"], s["scale"])
    return (out, *cache)


def work(case):
    op, Hkv, D = case["op"], case["Hkv"], case["D"]
    if op.startswith("rotate"):
        T, heads = case["B"] * case["S"], case["Hq"] + Hkv
        once = {"bytes": T * heads * D * 4 + 4 * T + 4 * case["R"], "flops": 3 * T * heads * case["R"]}
        return once if op == "rotate" else {x: 2 * y for x, y in once.items()}
    block = case["block"]
    if op in ("store", "load"):
        T = case["T"]
        return {"bytes": 2 * T * Hkv * 3 * D + 2 * Hkv * -(-T // block) + 8 * T, "flops": 4 * T * Hkv * D}
    B, Hq, page = case["B"], case["Hq"], case["page"]
    lens = _spread(case["low"], case["high"], B)
    moved = 2 * Hkv * (sum(lens) * D + sum(-(-x // block) for x in lens)) + 4 * B * Hq * D + 4 * B + 4 * sum(_pages(x, page) for x in lens)
    if case["lse"]:
        moved += 4 * B * Hq
    if op == "step":
        moved += 4 * B * Hkv * D + 8 * B  # the new rows come in 16 bits and go to the pool in 8
    return {"bytes": moved, "flops": 4 * sum(lens) * Hq * D}


def _told(pages, scales):
    """A pool's values in 64 bits, by token: [pages * page, Hkv, D]."""
    n, Hkv, page, D = pages.shape
    raw = scales.view(torch.uint8).double()
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=raw.device), raw - 127)
    scale = scale.masked_fill(raw == 255, math.nan).repeat_interleave(page // scales.shape[2], 2)
    return (pages.double() * scale[..., None]).transpose(1, 2).reshape(n * page, Hkv, D)


def exact(case, seed):
    """The definitions, token by token or request by request, in 64 bits; None for what is whole numbers or decided by rounding."""
    s = prepare(case, seed)
    op, D, Hkv = case["op"], case["D"], case["Hkv"]
    if op.startswith("rotate"):
        R = case["R"]
        at = s["positions"].double()[:, None, :, None] * s["frequencies"]
        wave = torch.polar(torch.full_like(at, s["magnitude"]), at)  # a rotation is a product of complex numbers

        def turned(x, by):
            x = x.detach().double()
            if case["pairs"] == "halves":
                z = torch.complex(x[..., : R // 2].contiguous(), x[..., R // 2: R].contiguous()) * by
                y = torch.cat((z.real, z.imag), -1)
            else:
                y = torch.view_as_real(torch.view_as_complex(x[..., :R].reshape(*x.shape[:3], R // 2, 2)) * by).flatten(-2)
            return torch.cat((y, x[..., R:]), -1)

        out = turned(s["q"], wave), turned(s["k"], wave)
        return out if op == "rotate" else (*out, turned(s["dq"], wave.conj()), turned(s["dk"], wave.conj()))
    if op == "store":
        if case["held"] == "int8" or case["block"] > 1:
            return None
        # before its rounding to a code of 4 bits, a value is the given one over its row's scale
        found = {}
        for x in "kv":
            codes, scales = s[x + "_pages"].double(), s[x + "_scales"].double()
            new = s["new_" + x][0].transpose(0, 1).double()
            scale = torch.pow(2.0, torch.ceil(torch.log2(new.abs().amax(-1) / 448)))
            at, inside = s["slots"] // case["page"], s["slots"] % case["page"]
            codes[at, :, inside], scales[at, :, inside] = new / scale[..., None], scale
            found[x] = codes, scales
        return found["k"][0], found["v"][0], found["k"][1], found["v"][1]
    if op == "load":
        return tuple(_told(s[x + "_pages"], s[x + "_scales"])[s["slots"]].transpose(0, 1)[None] for x in "kv")
    page = case["page"]
    if op == "step":
        # rounding decides what the newest row becomes: it is stored as the plain form stores it
        for x in "kv":
            _store(s[x + "_pages"], s[x + "_scales"], s["new_" + x], s["slots"], case["held"])
    B, Hq = case["B"], case["Hq"]
    lens, table = s["lengths"].tolist(), s["block_table"].long()
    out = torch.zeros(B, Hq, 1, D, dtype=torch.float64, device=table.device)
    lse = torch.full((B, Hq, 1), -math.inf, dtype=torch.float64, device=table.device)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        mine = table[b, : _pages(n, page)]
        k, v = (_told(s[x + "_pages"].view(torch.uint8)[mine].view(s[x + "_pages"].dtype),
                      s[x + "_scales"].view(torch.uint8)[mine].view(torch.float8_e8m0fnu))[:n].transpose(0, 1) for x in "kv")
        x = torch.einsum("hgd,hnd->hgn", s["q"][b, :, 0].double().view(Hkv, -1, D), k) * s["scale"]
        lse[b, :, 0] = torch.logsumexp(x, -1).view(-1)
        out[b, :, 0] = torch.einsum("hgn,hnd->hgd", torch.softmax(x, -1), v).reshape(Hq, D)
    if op == "step":
        return out, None, None, None, None
    return (out, lse) if case["lse"] else out
