# SPDX-License-Identifier: Apache-2.0
"""K8, storing with several tokens to a scale: tokens of one block anywhere in a call (GPU)."""
import math

import pytest
import torch

from kotflash_b200 import append_paged_kv8
from oracle import paged8_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _store(codes, exps, new, slots, held):
    """The definition, block by block: the largest magnitude of all of the
    call's rows, joined by the block's own scale if it has rows before the first
    of them, which are then rounded again; all rows under that scale."""
    pages, heads, page, d = codes.shape
    block = page // exps.shape[2]
    rows = new.double().transpose(1, 2).reshape(-1, heads, d)
    found = {}
    for t, s in enumerate(slots):
        if 0 <= s < pages * page:
            found.setdefault(s // block, []).append(t)
    for b, tokens in found.items():
        at, base = b * block // page, b * block % page
        first = min(slots[t] % block for t in tokens)
        for h in range(heads):
            x = rows[tokens, h]
            e = oracle.exponent(float("nan") if torch.isnan(x).any() else x.abs().max().item(), held)
            if first:
                was = exps[at, h, base // block].item()
                e = math.nan if math.isnan(e) or math.isnan(was) else max(e, was)
                kept = slice(base, base + first)
                if math.isnan(e):
                    codes[at, h, kept] = 0
                elif e > was:
                    codes[at, h, kept] = oracle.round_code(codes[at, h, kept] * 2.0 ** (was - e), held)
            exps[at, h, base // block] = e
            for t, y in zip(tokens, x):
                codes[at, h, base + slots[t] % block] = 0 if math.isnan(e) else oracle.round_code(y * 2.0 ** -e, held)


def _pool(n, heads, page, d, block, held, seed):
    g = torch.Generator().manual_seed(seed)
    top = oracle.LARGEST[held]
    codes = oracle.round_code((torch.randn(n, heads, page, d, generator=g, dtype=torch.float64) * top / 4).clamp(-top, top), held)
    exps = torch.randint(-9, -4, (n, heads, page // block), generator=g).double()
    raw = torch.full((n, heads, page, -(-d // 16) * 16), 0x7f, dtype=torch.uint8, device="cuda").view(oracle.FORMATS[held])[..., :d]
    raw.copy_(codes.float().cuda().to(raw.dtype))
    return codes, exps, raw, oracle.bytes_of(exps).cuda().view(torch.float8_e8m0fnu)


def _orders(page, block, n, seed):
    """Slots of one call: what should go to one block, apart in many ways."""
    g = torch.Generator().manual_seed(seed)
    every = torch.randperm(n * page, generator=g).tolist()
    runs = [every[0] // page * page + x for x in range(page)]
    half = max(1, page // 2)
    yield "shuffled", every[: min(len(every), 300)]
    yield "backwards", sorted(every[: min(len(every), 150)], reverse=True)
    yield "two halves, the later first", runs[half:] + [every[0] // page * page + page if every[0] // page < n - 1 else -1] + runs[:half]
    yield "holes", [s if i % 3 else -1 for i, s in enumerate(runs)] + [-1] * 40 + [s for i, s in enumerate(runs) if i % 3 == 0]
    yield "one token of each page, then another", [p * page + block // 2 for p in range(n)] + [p * page + block - 1 for p in range(n)]


@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,heads,d,page,block", [
    (BF16, 1, 64, 16, 16), (F16, 3, 72, 24, 8), (BF16, 2, 128, 64, 64), (F16, 8, 16, 4, 2), (BF16, 1, 40, 256, 128), (F16, 5, 128, 32, 4),
])
def test_tokens_of_a_block_determine_its_scale_together(held, dtype, heads, d, page, block):
    n = 12
    for i, (name, slots) in enumerate(_orders(page, block, n, page + d)):
        kc, ke, kp, ks = _pool(n, heads, page, d, block, held, 1 + i)
        vc, ve, vp, vs = _pool(n, heads, page, d, block, held, 50 + i)
        g = torch.Generator(device="cuda").manual_seed(i)
        size = torch.exp2(torch.randint(-12, 8, (2, 1, heads, len(slots), 1), device="cuda", generator=g).float())
        new = (torch.randn(2, 1, heads, len(slots), d, device="cuda", generator=g) * size).to(dtype)
        new[0, 0, 0, len(slots) // 2, 3] = math.inf
        append_paged_kv8(kp, vp, ks, vs, new[0], new[1], torch.tensor(slots, device="cuda"))
        for codes, exps, pages, scales, rows in ((kc, ke, kp, ks, new[0]), (vc, ve, vp, vs, new[1])):
            _store(codes, exps, rows.cpu(), slots, held)
            assert torch.equal(scales.cpu().view(torch.uint8), oracle.bytes_of(exps)), name
            assert torch.equal(pages.cpu().double(), codes), name


@pytest.mark.parametrize("held", ["e4m3", "int8"])
def test_runs_of_one_block_far_apart(held):
    """The parts of a block at both ends of a call of 20000 tokens, as a padded batch brings them."""
    page, block, heads, d, n = 64, 32, 2, 64, 330
    slots = [5 * page + i for i in range(3, 20)] + list(range(10 * page, 10 * page + 19000)) + [-1] * 900 \
        + [5 * page + i for i in range(20, 32)] + [5 * page + 1, 6 * page + 40] + list(range(7 * page + 32, 7 * page + 64))
    kc, ke, kp, ks = _pool(n, heads, page, d, block, held, 1)
    vc, ve, vp, vs = _pool(n, heads, page, d, block, held, 2)
    new = torch.randn(2, 1, heads, len(slots), d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    new[:, :, :, -40:] *= 50
    append_paged_kv8(kp, vp, ks, vs, new[0], new[1], torch.tensor(slots, device="cuda"))
    for codes, exps, pages, scales, rows in ((kc, ke, kp, ks, new[0]), (vc, ve, vp, vs, new[1])):
        _store(codes, exps, rows.cpu(), slots, held)
        assert torch.equal(scales.cpu().view(torch.uint8), oracle.bytes_of(exps))
        assert torch.equal(pages.cpu().double(), codes)


@pytest.mark.parametrize("held,dtype,page,block", [("e4m3", BF16, 32, 2), ("int8", F16, 48, 16), ("e4m3", F16, 64, 32), ("int8", BF16, 128, 128)])
def test_long_calls(held, dtype, page, block):
    """Calls long enough for thread blocks of their own for runs that do not fill
    their block: whole blocks, parts of blocks, and parts of one block apart."""
    heads, d, n = 3, 24, 3200 // page
    every = [p * page + i for p in torch.randperm(n, generator=torch.Generator().manual_seed(page)).tolist() for i in range(page)]
    cuts = [every[:700], every[705:1500], every[2011:], every[1507:2003]]  # some rows are not written
    apart = [x for c in cuts for x in (c[5:], c[:5])]
    g = torch.Generator(device="cuda").manual_seed(block)
    for slots in (sum(cuts, []), sum(apart, []), sum(cuts, [])[::-1]):
        assert len(slots) >= 2048
        kc, ke, kp, ks = _pool(n, heads, page, d, block, held, 1)
        vc, ve, vp, vs = _pool(n, heads, page, d, block, held, 2)
        new = (torch.randn(2, 1, heads, len(slots), d, device="cuda", generator=g) * 3).to(dtype)
        append_paged_kv8(kp, vp, ks, vs, new[0], new[1], torch.tensor(slots, device="cuda"))
        for codes, exps, pages, scales, rows in ((kc, ke, kp, ks, new[0]), (vc, ve, vp, vs, new[1])):
            _store(codes, exps, rows.cpu(), slots, held)
            assert torch.equal(scales.cpu().view(torch.uint8), oracle.bytes_of(exps))
            assert torch.equal(pages.cpu().double(), codes)
