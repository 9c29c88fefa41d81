# SPDX-License-Identifier: Apache-2.0
"""K9 over pools whose rows have gaps or whose pages fill no whole lines: the
results of dense pools, from memory that ends with the last row (GPU)."""
import pytest
import torch

from kotflash_b200 import append_paged_kv8, paged_attention8

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _at_the_end(shape, pitch, dtype):
    """A pool with rows `pitch` bytes apart whose last row ends where its allocation does."""
    n, heads, page, d = shape
    row = -(-d // 16) * 16
    size = ((n * heads * page) - 1) * pitch + row
    raw = torch.full((32 << 20,), 0x7f, dtype=torch.uint8, device="cuda")
    return raw.view(dtype).as_strided(shape, (heads * page * pitch, page * pitch, pitch, 1), raw.numel() - size)


@pytest.mark.parametrize("held", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype,hq,hkv,d,page,gap", [
    (F16, 17, 1, 24, 16, 16), (BF16, 4, 2, 72, 32, 32), (BF16, 40, 1, 64, 64, 16), (F16, 8, 8, 128, 16, 48), (BF16, 12, 1, 40, 3, 0),
    (F16, 6, 3, 16, 4, 0), (BF16, 64, 1, 104, 5, 16), (BF16, 16, 1, 120, 1, 0), (F16, 24, 2, 56, 128, 16), (BF16, 2, 2, 88, 100, 0),
])
@pytest.mark.parametrize("fused", [False, True])
def test_rows_with_gaps_at_the_end_of_memory(held, dtype, hq, hkv, d, page, gap, fused):
    """Rows with gaps lie otherwise in a tile, so sums may run in another order:
    a 32-bit evaluation each (n and D roundings of 2^-23 of scores up to 2^4 and of weights), rounded
    once each, so within one step of the output's type, 2^-10 or 2^-7, and 2^-12 of the largest value."""
    lens = [1, 37, 300]
    n = sum(-(-x // page) for x in lens) + 1
    pitch = -(-d // 16) * 16
    k = _at_the_end((n, hkv, page, d), pitch + gap, held)
    v = _at_the_end((n, hkv, page, d), pitch + gap, held)
    ks, vs = (torch.zeros(n, hkv, page, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
    order = torch.randperm(n - 1, generator=torch.Generator().manual_seed(n)).tolist() + [n - 1]
    order.reverse()                                   # the pool's last page is the first request's
    table = torch.full((3, max(-(-x // page) for x in lens)), -1, dtype=torch.int32)
    for b, x in enumerate(lens):
        for j in range(-(-x // page)):
            table[b, j] = order.pop(0)
    table = table.cuda()
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(d)
    rows = torch.randn(2, 1, hkv, n * page, d, device="cuda", generator=g).to(dtype)
    append_paged_kv8(k, v, ks, vs, rows[0], rows[1], torch.arange(n * page, device="cuda"))
    q = torch.randn(3, hq, 1, d, device="cuda", generator=g).to(dtype)
    new = {}
    if fused:
        slots = [int(table[b, (x - 1) // page]) * page + (x - 1) % page for b, x in enumerate(lens)]
        new = dict(new_k=torch.randn(3, hkv, 1, d, device="cuda", generator=g).to(dtype), new_v=torch.randn(3, hkv, 1, d, device="cuda", generator=g).to(dtype),
                   slots=torch.tensor(slots, device="cuda"))
    out, lse = paged_attention8(q, k, v, ks, vs, table, lengths, return_lse=True, **new)
    # the same rows in pages of 16 without gaps, one request after another
    kd, vd = (x.float().double() * torch.exp2(s.view(torch.uint8).double() - 127)[..., None] for x, s in ((k, ks), (v, vs)))
    for b, x in enumerate(lens):
        at = torch.arange(x, device="cuda")
        pages, inside = table[b].long()[at // page], at % page
        kb, vb = kd[pages, :, inside].transpose(0, 1), vd[pages, :, inside].transpose(0, 1)
        score = q[b, :, 0].double().view(hkv, -1, d) @ kb.transpose(1, 2) * d ** -0.5
        want = (torch.softmax(score, -1) @ vb).reshape(hq, 1, d)
        step = 2.0 ** -10 if dtype == F16 else 2.0 ** -7
        assert ((out[b].double() - want).abs() <= step * want.abs() + 2.0 ** -12 * vb.abs().max()).all()
        assert (lse[b, :, 0].double() - torch.logsumexp(score, -1).reshape(hq)).abs().max() <= 2.0 ** -14
