# SPDX-License-Identifier: Apache-2.0
"""K9, attention over the 8-bit paged cache: how exactly its weights are held and summed (GPU)."""
import math

import pytest
import torch

from kotflash_b200 import paged_attention8

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _pool(codes, exponents, held):
    """Codes [pages, page, D] and exponents [pages, page] of one KV head, rows on 16 bytes."""
    n, page, d = codes.shape
    raw = torch.zeros(n, 1, page, -(-d // 16) * 16, dtype=torch.uint8, device="cuda").view(FORMATS[held])[..., :d]
    raw.copy_(codes[:, None].to(FORMATS[held]))
    return raw, (exponents + 127).to(torch.uint8)[:, None].contiguous().view(torch.float8_e8m0fnu)


@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,d", [(8, 64), (8, 128), (6, 72), (16, 32), (24, 128), (64, 64)])
@pytest.mark.parametrize("n", [2, 3, 7, 20])
def test_outputs_are_a_32_bit_evaluation_rounded_once(held, dtype, hq, d, n):
    """Scores are one product each, |x| < 8 in base 2, so off by 2^-20 with all
    that scales them and a base-2 exponential (2^-22 of a weight); weights are
    held to 2^-20, n <= 20 of them and their products summed with fewer than 32
    roundings of 2^-24 and as many of a truncating MMA (2^-23).  So O is off by 2^-17 of the largest
    |v| and then rounded to nearest: by half a step of the value's binade
    (fp16: of its subnormals' at the least)."""
    g = torch.Generator(device="cuda").manual_seed(n + d)
    b, page = 40, 32
    codes = torch.randint(-60, 61, (2, b, page, d), device="cuda", generator=g).to(FORMATS[held]).double()
    exps = torch.stack((torch.full((b, page), -4, device="cuda"), torch.full((b, page), -7, device="cuda")))
    q = torch.zeros(b, hq, 1, d, device="cuda", dtype=dtype)
    q[:, torch.arange(hq), 0, torch.arange(hq) % d] = 1  # a column of K each
    q = q * torch.tensor([1.0, -1.5, 0.75, 1.875], device="cuda", dtype=dtype).repeat(hq)[:hq].view(1, hq, 1, 1)
    (kp, ks), (vp, vs) = _pool(codes[0], exps[0], held), _pool(codes[1], exps[1], held)
    table = torch.arange(b, dtype=torch.int32, device="cuda")[:, None].contiguous()
    lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
    out, lse = paged_attention8(q, kp, vp, ks, vs, table, lengths, scale=math.log(2), return_lse=True)
    k, v = codes[0, :, :n] / 16, codes[1, :, :n] / 128
    x = torch.einsum("bhd,bnd->bhn", q[:, :, 0].double(), k)
    assert x.abs().max() < 8
    w = torch.exp2(x)
    want = (torch.einsum("bhn,bnd->bhd", w, v) / w.sum(-1, keepdim=True))[:, :, None]
    bits, least = (11, -14) if dtype == F16 else (8, -126)
    half = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** least))) - bits)
    over = ((out.double() - want).abs() - half).max().item()
    bound = 2.0 ** -17 * v.abs().max().item()
    assert over <= bound, f"{over:.3e} past half a step, bound {bound:.3e}"
    assert (lse.double() - torch.log(w.sum(-1))[..., None]).abs().max().item() <= 2.0 ** -17 + 8 * 2.0 ** -22


@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("n,d,hq", [(64, 128, 1), (64, 128, 40), (500, 64, 2), (2000, 32, 24), (131072, 64, 1), (131072, 64, 16), (30000, 104, 64)])
@pytest.mark.parametrize("lead", [-20, 7, 18, 30])
def test_keys_without_a_value_beside_one_of_the_largest(held, n, d, hq, lead):
    """The scales' whole range: one key whose V has the largest exponent, 60,
    all others zeros, which have the smallest, wherever the one stands.  Scores
    are exact but for their scaling, 2^-22 of at most 30, and enter a weight by
    a base-2 exponential (2^-22): 2^-17 of a weight or less; sums of n equal
    ones as in any batch."""
    page, top = 16, {"e4m3": 448.0, "int8": 127.0}[held]
    pages = -(-n // page)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).to(torch.int32).cuda()[None]
    q = torch.zeros(1, hq, 1, d, device="cuda", dtype=BF16)
    q[..., 0] = 1
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    others = (n - 1) * 2.0 ** -lead
    bound = 2.0 ** -17 + (n / 16 + 64) * 2.0 ** -23
    for where in (0, 31, n // 2, n - 1):
        at, row = int(table[0, where // page]), where % page
        k, v = (torch.zeros(pages, page, d, device="cuda") for _ in range(2))
        ke, ve = torch.zeros(pages, page, device="cuda"), torch.full((pages, page), -60.0, device="cuda")
        k[at, row, 0], v[at, row], ve[at, row] = lead, top, 60
        (kp, ks), (vp, vs) = _pool(k, ke, held), _pool(v, ve, held)
        out, lse = paged_attention8(q, kp, vp, ks, vs, table, lengths, scale=math.log(2), return_lse=True)
        want = top * 2.0 ** 60 / (1 + others)
        err = (out.double() / want - 1).abs().max().item()
        assert err <= 2.0 ** -8 + 2 * bound, f"key {where}: off by {err:.3e} of the value"
        want = lead * math.log(2) + math.log1p(others)
        err = (lse.double() - want).abs().max().item()
        assert err <= bound + abs(want) * 2.0 ** -22, f"key {where}: LSE off by {err:.3e}"
