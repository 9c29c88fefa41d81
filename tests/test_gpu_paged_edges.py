# SPDX-License-Identifier: Apache-2.0
"""The paged KV cache at its edges (GPU)."""
import math

import pytest
import torch

from kotflash_b200 import paged_attention

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# ---------------------------------------------------------------- one dominant key

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq", [1, 40])                       # four teams that share the keys, and one
@pytest.mark.parametrize("lead", [12.5, 20.0, 24.5, 25.25, 30.0])
@pytest.mark.parametrize("place", [5, 20000, 32767])
def test_the_rest_of_a_row_that_one_key_dominates(dtype, hq, lead, place):
    """One of 32768 keys lies 2^lead above the others, which are all alike, so
    O and the LSE follow from a count.  Enough requests that a block takes
    whole rows, so that the weights of one reference fill a team's keys.

    Bounds: a weight is off by 2^-16 of itself (two 16-bit parts) and its score
    (30 in base 2 at most, 2^-19 of the weight); in fp16 also by the smallest
    parts, 2^-35 of the row's largest weight.  Sums run over n / 16 products of
    16 keys, each step off by 2^-23 of the sum.  The output is rounded once."""
    n, d, page, b = 32768, 64, 64, 300
    k = torch.zeros(n // page, 1, page, d, device="cuda", dtype=dtype)
    k[place // page, 0, place % page, 0] = lead
    q = torch.zeros(b, hq, 1, d, device="cuda", dtype=dtype)
    q[..., 0] = 1
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(b, -1).contiguous()
    lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
    others = (n - 1) * 2.0 ** -lead
    hold = 2.0 ** -16 + 2.0 ** -19 + (n / 16 + 64) * 2.0 ** -23
    for at_peak in (0.0, 1.0):
        v = torch.ones_like(k)
        v[place // page, 0, place % page] = at_peak
        out, lse = paged_attention(q, k, v, table, lengths, scale=math.log(2), return_lse=True)
        want = (at_peak + others) / (1 + others)
        bound = UNIT[dtype] * want + 2.0 ** -24 + 2 * want * hold + n * 2.0 ** -35
        err = (out.double() - want).abs().max().item()
        assert err <= bound, f"off by {err:.3e}, bound {bound:.3e}, value {want:.3e}"
        want = lead * math.log(2) + math.log1p(others)
        err = (lse.double() - want).abs().max().item()
        assert err <= hold + want * 2.0 ** -22, f"LSE off by {err:.3e}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq", [1, 40])
@pytest.mark.parametrize("lead", [20.0, 22.5, 23.5, 24.25, 25.25, 26.0])
def test_many_small_weights_beside_a_large_sum(dtype, hq, lead):
    """131072 keys beside one that leads by 2^lead, all values 1: O = 1.

    Bounds: as above, with the large sum from the first tile on."""
    n, d, page, b = 131072, 64, 64, 300
    k = torch.zeros(n // page, 1, page, d, device="cuda", dtype=dtype)
    k[0, 0, 5, 0] = lead
    q = torch.zeros(b, hq, 1, d, device="cuda", dtype=dtype)
    q[..., 0] = 1
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(b, -1).contiguous()
    lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
    out, lse = paged_attention(q, k, torch.ones_like(k), table, lengths, scale=math.log(2), return_lse=True)
    hold = 2.0 ** -16 + 2.0 ** -19 + (n / 16 + 64) * 2.0 ** -23
    assert (out.double() - 1).abs().max().item() <= UNIT[dtype] + hold
    want = lead * math.log(2) + math.log1p((n - 1) * 2.0 ** -lead)
    assert (lse.double() - want).abs().max().item() <= hold + want * 2.0 ** -22
