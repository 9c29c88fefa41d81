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
