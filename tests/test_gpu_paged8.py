# SPDX-License-Identifier: Apache-2.0
"""K8/K9, the paged KV cache in 8 bits, against the 64-bit oracle (GPU)."""
import math

import pytest
import torch

from kotflash_b200 import PagedKVCache8, append_paged_kv8, apply_rotary, paged_attention8, read_paged_kv8, rotary_frequencies
from oracle import paged8_oracle as oracle8
from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}  # unit roundoff of the output's type


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def _codes(n, hkv, page, d, held, seed, block=1, low=-9, high=-5):
    """A pool of codes (float64, CPU) and exponents, as rows of normal values have them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, hkv, page, d, generator=g, dtype=torch.float64)
    x = oracle8.round_code((x * (100 if held == "e4m3" else 35)).clamp(-oracle8.LARGEST[held], oracle8.LARGEST[held]), held)
    return x, torch.randint(low, high + 1, (n, hkv, page // block), generator=g).double()


def _pool(codes, exps, held, pad=16):
    """The pool on the GPU, rows on 16 bytes, with junk between them."""
    n, hkv, page, d = codes.shape
    raw = torch.full((n, hkv, page, -(-d // pad) * pad), 0x7f, dtype=torch.uint8, device="cuda").view(oracle8.FORMATS[held])
    raw[..., :d] = codes.float().cuda().to(oracle8.FORMATS[held])
    return raw[..., :d], oracle8.bytes_of(exps).cuda().view(torch.float8_e8m0fnu)


def _same(pages, scales, codes, exps):
    raw = oracle8.bytes_of(exps)
    assert torch.equal(scales.cpu().view(torch.uint8), raw), "scales differ"
    assert torch.equal(pages.cpu().double(), codes), "codes differ"


# ---------------------------------------------------------------- storing

def _awkward(shape, dtype, seed):
    """Rows over the whole range of a type: magnitudes from the smallest to the
    largest, ties, zeros, borders of both formats, infinities and NaN."""
    x = _rand(shape, torch.float32, seed)
    x = x * torch.exp2(torch.randint(-30, 15, shape[:3], device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).float())[..., None]
    x = x.to(dtype)
    rows = x.view(-1, shape[-1])  # contiguous
    n = rows.shape[0]
    special = [0.0, 448.0, 449.0, 127.0, 127.5, 1.0, 255.0, torch.finfo(dtype).max, torch.finfo(dtype).tiny / 4, 896.0, math.inf, math.nan, -math.inf]
    for i, value in enumerate(special):
        if i < n:
            rows[i] = torch.linspace(-1, 1, shape[-1], device="cuda").to(dtype)
            rows[i] *= 0 if value == 0 else 0.5
            rows[i, i % shape[-1]] = value
    if n > 16:
        rows[14] = (torch.arange(shape[-1], device="cuda") % 64 + 0.5).to(dtype)   # ties of int8 under a scale of 1
        rows[14, 0] = 127
        rows[15] = (torch.arange(shape[-1], device="cuda") + 16.0 + 17 * (torch.arange(shape[-1], device="cuda") % 2)).to(dtype)
    return x


@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hkv,d,page,block,T", [
    (1, 128, 16, 1, 1), (8, 128, 16, 1, 300), (2, 72, 24, 1, 77), (3, 16, 5, 1, 33), (1, 40, 1, 1, 9), (16, 64, 64, 1, 50),
    (2, 128, 16, 16, 100), (3, 72, 24, 8, 61), (1, 16, 256, 128, 400), (2, 104, 32, 32, 90), (1, 64, 4, 2, 31), (4, 96, 64, 64, 70),
])
def test_stores_what_the_oracle_stores(held, dtype, hkv, d, page, block, T):
    n = 2 * -(-T // page) + 6
    g = torch.Generator().manual_seed(T + d)
    order = torch.randperm(n, generator=g).tolist()
    # runs behind rows that are there already, in pages of their own, with refused tokens and slots outside between
    slots, at = [], 0
    while len(slots) < T:
        size = min(T - len(slots), int(torch.randint(1, 2 * page + 2, (1,), generator=g)))
        begin = int(torch.randint(0, page, (1,), generator=g))
        for i in range(begin, begin + size):
            if at + i // page < n:
                slots.append(order[at + i // page] * page + i % page)
        at += -(-(begin + size) // page)
        if at >= n:
            slots += [-1, n * page, 2 ** 40, -7][: T - len(slots)]
            break
        if len(slots) < T:
            slots.append(-1)
    slots = (slots + [-1] * T)[:T]
    kc, ke = _codes(n, hkv, page, d, held, 1, block)
    vc, ve = _codes(n, hkv, page, d, held, 2, block)
    (kp, ks), (vp, vs) = _pool(kc, ke, held), _pool(vc, ve, held)
    nk, nv = _awkward((1, hkv, T, d), dtype, 3), _awkward((1, T, hkv, d), dtype, 4).transpose(1, 2)
    append_paged_kv8(kp, vp, ks, vs, nk, nv, torch.tensor(slots, dtype=torch.int64, device="cuda"))
    oracle8.store(kc, ke, nk.cpu(), slots, held)
    oracle8.store(vc, ve, nv.cpu(), slots, held)
    _same(kp, ks, kc, ke)
    _same(vp, vs, vc, ve)
    if d % 16:  # what lies between rows stays
        pitch = kp.stride(2)
        between = torch.as_strided(kp, (n, hkv, page, pitch - d), kp.stride(), d)
        assert (between.view(torch.uint8) == 0x7f).all()


@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [2, 16, 64])
def test_tokens_one_by_one_raise_a_blocks_scale(held, block):
    """A block filled token by token, magnitudes rising and falling, one row not
    finite in one head, then begun anew."""
    page, hkv, d = 64, 3, 48
    kc, ke = _codes(4, hkv, page, d, held, 5, block)
    vc, ve = _codes(4, hkv, page, d, held, 6, block)
    (kp, ks), (vp, vs) = _pool(kc, ke, held), _pool(vc, ve, held)
    g = torch.Generator().manual_seed(7)
    for i in list(range(page)) + [0, 1]:
        scale = 2.0 ** int(torch.randint(-12, 12, (1,), generator=g))
        nk, nv = _rand((1, hkv, 2, d), BF16, 100 + i, scale), _rand((1, hkv, 2, d), BF16, 200 + i)
        if i == 37:
            nk[0, 1, 0, 5] = math.nan
        slots = [2 * page + i, 0 * page + i]
        append_paged_kv8(kp, vp, ks, vs, nk, nv, torch.tensor(slots, device="cuda"))
        oracle8.store(kc, ke, nk.cpu(), slots, held)
        oracle8.store(vc, ve, nv.cpu(), slots, held)
    _same(kp, ks, kc, ke)
    _same(vp, vs, vc, ve)


# ---------------------------------------------------------------- reading back

@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hkv,d,page,block,T", [(1, 128, 16, 1, 1), (8, 128, 16, 16, 333), (3, 72, 24, 8, 50), (2, 16, 5, 1, 1000), (5, 104, 7, 1, 64)])
def test_reads_what_the_codes_stand_for(held, dtype, hkv, d, page, block, T):
    n = 40
    kc, ke = _codes(n, hkv, page, d, held, 1, block, -30, 12)
    vc, ve = _codes(n, hkv, page, d, held, 2, block, -16, 4)
    ke[3, 0, 0] = math.nan
    (kp, ks), (vp, vs) = _pool(kc, ke, held), _pool(vc, ve, held)
    slots = torch.randint(-2, n * page + 2, (T,), generator=torch.Generator().manual_seed(1))
    slots[0] = 3 * page
    k, v = read_paged_kv8(kp, vp, ks, vs, slots.cuda(), dtype=dtype)
    assert k.shape == v.shape == (1, hkv, T, d) and k.dtype == dtype
    inside = (slots >= 0) & (slots < n * page)
    at = slots.clamp(0, n * page - 1)
    for got, codes, exps in ((k, kc, ke), (v, vc, ve)):
        want = oracle8.values(codes, exps)[at // page, :, at % page].to(dtype)  # [T, Hkv, D], exact or rounded once
        want = torch.where(inside[:, None, None], want, torch.zeros((), dtype=dtype)).transpose(0, 1)[None]
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.cpu()), torch.nan_to_num(want))


def test_what_is_read_is_stored_as_it_was():
    """Stored, read and stored again: the same codes, in both types and formats."""
    for held in ("e4m3", "int8"):
        for dtype in (F16, BF16):
            x = _rand((1, 4, 50, 64), dtype, 1)
            slots = torch.arange(50, device="cuda")
            (kp, ks), (vp, vs) = _pool(*_codes(4, 4, 16, 64, held, 1), held), _pool(*_codes(4, 4, 16, 64, held, 2), held)
            append_paged_kv8(kp, vp, ks, vs, x, x, slots)
            before = kp.view(torch.uint8).clone(), ks.view(torch.uint8).clone()
            k, _ = read_paged_kv8(kp, vp, ks, vs, slots, dtype=dtype)
            # the error of a stored element
            top = x.abs().amax(-1, keepdim=True).double()
            off = (k.double() - x.double()).abs()
            assert (off <= (torch.maximum(x.double().abs() * 2.0 ** -4, top / 224 * 2.0 ** -10) if held == "e4m3" else top * 2.0 ** -7)).all()
            append_paged_kv8(kp, vp, ks, vs, k, k, slots)
            if held == "e4m3":  # (a largest value that was rounded up may take the next scale)
                assert torch.equal(read_paged_kv8(kp, vp, ks, vs, slots, dtype=dtype)[0], k)
            else:
                assert torch.equal(kp.view(torch.uint8), before[0]) and torch.equal(ks.view(torch.uint8), before[1])


# ---------------------------------------------------------------- attention

def _requests(lens, page, hkv, d, held, seed, block=1, spread=(-9, -5), extra_cols=1, spare=3):
    """Pools whose pages are handed out at random; rows that no request sees hold
    NaN codes and NaN scales, table entries past a request's pages junk."""
    g = torch.Generator().manual_seed(seed)
    held_pages = [-(-n // page) for n in lens]
    n_pages = sum(held_pages) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    cols = max(held_pages) + extra_cols
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    visible = torch.zeros(n_pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        for j in range(held_pages[b]):
            table[b, j] = order[at]
            visible[order[at], : min(page, n - j * page)] = True
            at += 1
        for j in range(held_pages[b], cols):
            table[b, j] = order[j % n_pages] if j % 2 else -1 if j % 4 else 2**31 - 1
    pools = []
    for i in range(2):
        codes, exps = _codes(n_pages, hkv, page, d, held, seed + 1 + i, block, *spread)
        pages, scales = _pool(codes, exps, held)
        junk = pages.view(torch.uint8)
        junk[~visible.cuda()[:, None, :, None].expand(junk.shape)] = 0x7f
        mine = visible.view(n_pages, page // block, block).any(-1)
        scales.view(torch.uint8)[~mine.cuda()[:, None].expand(scales.shape)] = 255
        pools.append((pages, scales, oracle8.values(codes, exps)))
    (kp, ks, kv), (vp, vs, vv) = pools
    return (kp, vp, ks, vs), kv, vv, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def _check(out, lse, q, kv, vv, table, lengths, scale, name):
    """Bounds.  A score in base 2 is a sum of D exact products in fp32 (D 2^-23
    sum |q_i k_i| scale log2 e, tensor cores truncating; bf16 queries are exact
    in fp16 to 2^-39 of the row's largest, less than that), scaled and shifted
    by V's exponent f, |f| <= 60 ((|x| + 60) 2^-23), and enters a weight by a
    base-2 exponential (2^-22).  A weight is cut to fp16, by 0 to 2^-10 of
    itself, that is by 2^-11 and 2^-11 more or less; O is divided by the sum of
    the cut ones, so the first part cancels and the second moves O by 2^-11 max
    |v - O| <= 2^-10 max |v|; or, of a small one, by 2^-36 of the largest
    weight, of n.  For fp16 queries what is cut off is a second part, off by
    2^-11 of its 2^-10: 2^-21 of a weight, 2^-20 of max |v|.  Products and weights are summed 16 at a time in fp32 over n
    keys, plus a handful of joins; the output is rounded once (u)."""
    eo, el, sizes = oracle.attention(q, kv, vv, table, lengths, scale)
    o = out.double().cpu()
    d = q.shape[-1]
    assert out.shape == q.shape and out.dtype == q.dtype
    for b, (prod, vmax, n) in enumerate(sizes):
        if n == 0:
            assert (o[b] == 0).all(), f"{name}: request {b} sees nothing"
            assert lse is None or (lse[b] == -math.inf).all()
            continue
        dx = prod * (d + 4) * 2.0 ** -23 + 60 * 2.0 ** -23 + 2.0 ** -22
        summed = (n / 16 + 64) * 2.0 ** -23
        err = (o[b] - eo[b]).abs()
        held = 2.0 ** -10 if q.dtype == BF16 else 2.0 ** -20
        bound = UNIT[q.dtype] * eo[b].abs() + vmax * (held + 2 * dx + summed + n * 2.0 ** -35) + 2.0 ** -24
        assert (err <= bound).all(), f"{name}: request {b} (n={n}) off by {err.max():.3e}, bound {bound.min():.3e}"
        if lse is not None:
            assert lse.shape == q.shape[:3] and lse.dtype == torch.float32
            el_b = (lse[b].double().cpu() - el[b]).abs().max().item()
            assert el_b <= dx + summed + el[b].abs().max().item() * 2.0 ** -22, f"{name}: LSE {b} off by {el_b}"


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500, 1999]


@pytest.mark.parametrize("hq,hkv,d,dtype,held,page,block", [
    (8, 2, 64, F16, "e4m3", 16, 1),
    (32, 8, 128, BF16, "e4m3", 16, 1),
    (4, 4, 128, F16, "int8", 64, 64),    # one row per KV head
    (6, 2, 72, BF16, "int8", 24, 8),     # pages that end inside a tile
    (8, 1, 104, F16, "e4m3", 5, 1),
    (12, 1, 128, BF16, "e4m3", 1, 1),    # two row tiles, one position per page
    (16, 1, 64, F16, "int8", 3, 1),
    (24, 1, 128, F16, "e4m3", 100, 4),   # a team of two warps
    (32, 1, 40, BF16, "int8", 8, 2),
    (40, 1, 128, BF16, "int8", 32, 1),   # a team of four
    (64, 1, 16, F16, "e4m3", 256, 128),
    (72, 1, 96, BF16, "e4m3", 16, 16),   # two row blocks
    (130, 2, 24, F16, "int8", 7, 1),
    (48, 1, 64, BF16, "e4m3", 128, 1),
    (24, 1, 56, BF16, "e4m3", 64, 1),
])
def test_ragged_batches_against_the_oracle(hq, hkv, d, dtype, held, page, block):
    cache, kv, vv, table, lengths = _requests(LENS, page, hkv, d, held, 11, block)
    q = _rand((len(LENS), hq, 1, d), dtype, 7, 1.5)
    out, lse = paged_attention8(q, *cache, table, lengths, return_lse=True)
    _check(out, lse, q, kv, vv, table, lengths, d ** -0.5, f"{hq},{hkv},{d},{held},{page}")
    assert torch.equal(out, paged_attention8(q, *cache, table, lengths))


@pytest.mark.parametrize("d", range(16, 129, 8))
@pytest.mark.parametrize("page", [2, 4, 8, 16, 32, 64])
def test_every_head_dim_and_tile_layout(d, page):
    lens = [33, 1, 150, 260]
    for hq, dtype, held in ((6, BF16, "e4m3"), (40, F16, "int8"), (24, BF16, "int8")):
        cache, kv, vv, table, lengths = _requests(lens, page, 2, d, held, 200 + d + page)
        q = _rand((len(lens), hq, 1, d), dtype, 201, 1.5)
        out, lse = paged_attention8(q, *cache, table, lengths, return_lse=True)
        _check(out, lse, q, kv, vv, table, lengths, d ** -0.5, f"layout {d},{page},{hq}")


@pytest.mark.parametrize("hq,hkv,d,dtype,held,page,lens", [
    (8, 2, 64, F16, "e4m3", 64, [30000, 12345]),         # few requests: many partials to join
    (4, 1, 128, BF16, "int8", 16, [20011]),
    (32, 1, 128, F16, "e4m3", 16, [5000, 1]),
    (64, 1, 64, BF16, "int8", 32, [9000]),
    (8, 8, 128, BF16, "e4m3", 16, [700] * 40),           # many units per block
    (8, 4, 96, F16, "e4m3", 16, [3001, 40, 2999]),
])
def test_long_and_many(hq, hkv, d, dtype, held, page, lens):
    cache, kv, vv, table, lengths = _requests(lens, page, hkv, d, held, 21)
    q = _rand((len(lens), hq, 1, d), dtype, 22, 1.5)
    out, lse = paged_attention8(q, *cache, table, lengths, return_lse=True)
    _check(out, lse, q, kv, vv, table, lengths, d ** -0.5, "long")


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30])
def test_scales_of_any_sign(scale):
    cache, kv, vv, table, lengths = _requests([70, 3, 0], 16, 2, 64, "e4m3", 31)
    q = _rand((3, 4, 1, 64), BF16, 32)
    out, lse = paged_attention8(q, *cache, table, lengths, scale=scale, return_lse=True)
    _check(out, lse, q, kv, vv, table, lengths, scale, "scale")


@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("hq", [2, 40])
def test_values_whose_scales_lie_far_apart(held, hq):
    """V's scales from 2^-60 to 2^60, K's over 2^12: weights carry them, so O is
    right to a part of the largest single contribution, which bounds it here."""
    n, d = 3000, 64
    cache, kv, vv, table, lengths = _requests([n], 16, 1, d, held, 41, 1, (-16, -4))
    vs = cache[3].view(torch.uint8)
    g = torch.Generator(device="cuda").manual_seed(3)
    vs.copy_(torch.randint(67, 188, vs.shape, generator=g, device="cuda", dtype=torch.uint8))
    vv = oracle8.values(cache[1].cpu().double(), oracle8.exps_of(cache[3]))
    vv = torch.nan_to_num(vv)
    q = _rand((1, hq, 1, d), F16, 42, 1.5).bfloat16()
    out, lse = paged_attention8(q, *cache, table, lengths, scale=0.05, return_lse=True)
    eo, el, sizes = oracle.attention(q, kv, vv, table, lengths, 0.05)
    # the sum of the contributions' magnitudes stands for max |v - O| of _check
    mag, _, _ = oracle.attention(q, kv, vv.abs(), table, lengths, 0.05)
    dx = sizes[0][0] * (d + 4) * 2.0 ** -23 + 60 * 2.0 ** -23 + 2.0 ** -22
    err = (out.double().cpu() - eo).abs()
    assert (err <= 2.0 ** -8 * eo.abs() + mag.amax(-1, keepdim=True) * (2.0 ** -10 + 2 * dx + 300 * 2.0 ** -23 + n * 2.0 ** -35)).all()
    assert (lse.double().cpu() - el).abs().max() <= dx + 300 * 2.0 ** -23 + el.abs().max() * 2.0 ** -22


@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("hq", [2, 40])
def test_keys_whose_values_are_zero_count(held, hq):
    """Rows of zeros, whose scale is the smallest, still weigh on the others."""
    cache, kv, vv, table, lengths = _requests([700, 33], 16, 1, 64, held, 45)
    slots = torch.tensor([int(table[b, p // 16]) * 16 + p % 16 for b, p in [(0, i) for i in range(0, 700, 3)] + [(1, 0)]], device="cuda")
    k, _ = read_paged_kv8(*cache, slots, dtype=BF16)
    append_paged_kv8(*cache, k, torch.zeros_like(k), slots)
    kv, vv = (oracle8.values(p.cpu().double().nan_to_num(), oracle8.exps_of(s).nan_to_num()) for p, s in ((cache[0], cache[2]), (cache[1], cache[3])))
    q = _rand((2, hq, 1, 64), F16, 46, 1.5)
    out, lse = paged_attention8(q, *cache, table, lengths, return_lse=True)
    _check(out, lse, q, kv, vv, table, lengths, 64 ** -0.5, "zeros")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq", [1, 40])
@pytest.mark.parametrize("lead", [0.0, 12.5, 20.0, 24.0])
def test_many_small_weights_beside_a_large_one(dtype, hq, lead):
    """65536 equal keys beside one that leads by 2^lead, all values 1 or the
    leader's 0.  Equal weights round alike, so O = 1 to the output's rounding
    and the sums'; with the leader at 0 a weight is off by 2^-11 of itself, or
    by 2^-36 of the leader's, which n of them add up to n 2^-36 of O."""
    n, d, page, b = 65536, 64, 64, 40
    held = "e4m3"
    codes = torch.zeros(n // page, 1, page, d, dtype=torch.float64)
    codes[7, 0, 5, 0] = 16 * lead
    kp, ks = _pool(codes, torch.full((n // page, 1, page), -4.0, dtype=torch.float64), held)
    lead = float(kp.double().max()) / 16
    q = torch.zeros(b, hq, 1, d, device="cuda", dtype=dtype)
    q[..., 0] = 1
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(b, -1).contiguous()
    lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
    others = (n - 1) * 2.0 ** -lead
    summed = 2.0 ** -19 + (n / 16 + 64) * 2.0 ** -23
    for at_peak in (0.0, 1.0):
        v = torch.full_like(codes, 8.0)
        v[7, 0, 5] = 8 * at_peak
        vp, vs = _pool(v, torch.full((n // page, 1, page), -3.0, dtype=torch.float64), held)
        out, lse = paged_attention8(q, kp, vp, ks, vs, table, lengths, scale=math.log(2), return_lse=True)
        want = (at_peak + others) / (1 + others)
        bound = UNIT[dtype] * want + 2.0 ** -24 + 2 * want * summed + (2.0 ** -11 * want + n * 2.0 ** -36 if at_peak == 0 else 0)
        err = (out.double() - want).abs().max().item()
        assert err <= bound, f"off by {err:.3e}, bound {bound:.3e}, value {want:.3e}"
        want = lead * math.log(2) + math.log1p(others)
        assert (lse.double() - want).abs().max().item() <= summed + want * 2.0 ** -22


@pytest.mark.parametrize("hq", [2, 24, 72])
def test_nan_where_it_is_seen_and_nowhere_else(hq):
    """A NaN scale of V makes its head's O NaN and leaves the LSE; one of K makes
    both NaN; a NaN code of V its column."""
    cache, kv, vv, table, lengths = _requests([300, 40, 500], 16, 2, 64, "e4m3", 51)
    q = _rand((3, 2 * hq, 1, 64), F16, 52)
    want, want_lse = paged_attention8(q, *cache, table, lengths, return_lse=True)
    spoiled = [x.clone() for x in cache]

    def at(b, p):
        return int(table[b, p // 16]), p % 16

    page, row = at(0, 299)
    spoiled[3].view(torch.uint8)[page, 0, row] = 255
    page, row = at(1, 20)
    spoiled[2].view(torch.uint8)[page, 1, row] = 255
    page, row = at(2, 0)
    spoiled[1].view(torch.uint8)[page, 1, row, 9] = 0x7f
    out, lse = paged_attention8(q, *spoiled, table, lengths, return_lse=True)
    nan = torch.zeros(3, 2, hq, 64, dtype=torch.bool, device="cuda")
    nan[0, 0] = nan[1, 1] = True
    nan[2, 1, :, 9] = True
    nan = nan.view(3, 2 * hq, 1, 64)
    assert torch.equal(torch.isnan(out), nan) and torch.equal(out[~nan], want[~nan])
    nan_lse = torch.zeros(3, 2, hq, dtype=torch.bool, device="cuda")
    nan_lse[1, 1] = True
    nan_lse = nan_lse.view(3, 2 * hq, 1)
    assert torch.equal(torch.isnan(lse), nan_lse)
    # the head whose V has no exponent at one key sums with another reference: twice _check's bound
    # of an LSE; all others are untouched
    _, el, sizes = oracle.attention(q, kv, vv, table, lengths, 64 ** -0.5)
    bound = sizes[0][0] * 68 * 2.0 ** -23 + 60 * 2.0 ** -23 + 2.0 ** -22 + (300 / 16 + 64) * 2.0 ** -23 + el[0].abs().max().item() * 2.0 ** -22
    assert (lse[0, :hq] - want_lse[0, :hq]).abs().max().item() <= 2 * bound
    nan_lse[0, :hq] = True
    assert torch.equal(lse[~nan_lse], want_lse[~nan_lse])


def test_pages_outside_the_pool_are_masked():
    cache, kv, vv, table, lengths = _requests([200, 333, 64], 16, 2, 128, "int8", 61)
    table[0, 3], table[1, 0], table[1, 7] = -1, 2**31 - 1, cache[0].shape[0]
    table[2, :] = -5
    q = _rand((3, 4, 1, 128), BF16, 62)
    out, lse = paged_attention8(q, *cache, table, lengths, return_lse=True)
    _check(out, lse, q, kv, vv, table, lengths, 128 ** -0.5, "holes")


def test_pools_with_any_strides():
    """Tokens outside heads, K and V laid out differently, scales as views."""
    lens, page, hkv, d = [130, 17], 16, 2, 64
    cache, kv, vv, table, lengths = _requests(lens, page, hkv, d, "e4m3", 71)
    kp = cache[0].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(cache[1].shape[0], hkv + 1, page, d + 16, device="cuda", dtype=torch.uint8).view(cache[1].dtype)
    vp = wide[:, 1:, :, 16:]
    vp.copy_(cache[1])
    both = torch.stack((cache[2].view(torch.uint8), cache[3].view(torch.uint8)), 1).view(torch.float8_e8m0fnu)
    q = _rand((2, 4, 3, d), BF16, 72)[:, :, 1:2]
    want = paged_attention8(q, *cache, table, lengths)
    _check(want, None, q, kv, vv, table, lengths, d ** -0.5, "dense")
    # (rows with gaps lie otherwise in a tile, so their sums run in another order)
    _check(paged_attention8(q, kp, vp, both[:, 0], both[:, 1], table, lengths), None, q, kv, vv, table, lengths, d ** -0.5, "strided")
    slots = torch.tensor([int(table[0, 0]) * page + 3, int(table[1, 0]) * page], device="cuda")
    for got, ref in zip(read_paged_kv8(kp, vp, both[:, 0], both[:, 1], slots, dtype=BF16), read_paged_kv8(*cache, slots, dtype=BF16)):
        assert torch.equal(got, ref)
    x = _rand((1, hkv, 2, d + 3), BF16, 73)[..., 3:]  # rows off 16 bytes
    append_paged_kv8(kp, vp, both[:, 0], both[:, 1], x, x, slots)
    append_paged_kv8(*cache, x.contiguous(), x.contiguous(), slots)
    for got, ref in ((kp, cache[0]), (vp, cache[1])):
        assert torch.equal(got.contiguous().view(torch.uint8), ref.contiguous().view(torch.uint8))
    assert torch.equal(both[:, 0].contiguous().view(torch.uint8), cache[2].view(torch.uint8))


@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (72, 16), (32, 64), (16, 128), (96, 8)])
def test_k_and_v_however_they_lie_to_one_another(d, page):
    """K before V, V before K, both in one buffer, side by side in every page, one
    pool as both, with different strides: the same values, so the same results."""
    lens, hkv = [300, 41, 900], 2
    cache, kv, vv, table, lengths = _requests(lens, page, hkv, d, "e4m3", 75)
    kp, vp, ks, vs = cache
    n, pitch = kp.shape[0], kp.stride(2)
    q = _rand((3, 6, 1, d), BF16, 76)
    want, want_lse = paged_attention8(q, *cache, table, lengths, return_lse=True)

    def blank(*shape):
        return torch.full((*shape, pitch), 0x7f, device="cuda", dtype=torch.uint8).view(kp.dtype)[..., :d]

    both = blank(2, n, hkv, page)
    for first, second in ((0, 1), (1, 0)):
        k, v = both[first], both[second]
        k.copy_(kp), v.copy_(vp)
        out, lse = paged_attention8(q, k, v, ks, vs, table, lengths, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    side = blank(n, 2, hkv, page)
    k, v = side[:, 1], side[:, 0]
    k.copy_(kp), v.copy_(vp)
    assert torch.equal(paged_attention8(q, k, v, ks, vs, table, lengths), want)
    wide = blank(n, hkv + 1, page)[:, 1:]                     # V with other strides than K
    wide.copy_(vp)
    assert torch.equal(paged_attention8(q, kp, wide, ks, vs, table, lengths), want)
    _check(paged_attention8(q, kp, kp, ks, ks, table, lengths), None, q, kv, kv, table, lengths, d ** -0.5, "one pool")


# ---------------------------------------------------------------- the append on the way

@pytest.mark.parametrize("hq,hkv,d,dtype,held,page,block", [
    (8, 2, 64, F16, "e4m3", 16, 1), (32, 8, 128, BF16, "int8", 16, 1), (6, 2, 72, BF16, "e4m3", 24, 1), (24, 1, 96, F16, "int8", 32, 1),
    (72, 1, 128, BF16, "e4m3", 64, 1), (130, 2, 24, F16, "e4m3", 7, 1), (40, 1, 64, BF16, "int8", 16, 1), (12, 4, 128, F16, "e4m3", 1, 1),
    (8, 2, 128, BF16, "e4m3", 16, 16), (24, 2, 72, F16, "int8", 24, 8), (72, 1, 64, BF16, "int8", 64, 4),
])
def test_the_fused_append_is_append_then_attend(hq, hkv, d, dtype, held, page, block):
    lens = [1, 16, 17, 300, 64, 65, 129, 2, 700, 0]
    b = len(lens)
    cache, kv, vv, table, lengths = _requests(lens, page, hkv, d, held, 81, block)
    q, nk, nv = _rand((b, hq, 1, d), dtype, 82), _rand((b, 1, hkv, d), dtype, 83).transpose(1, 2), _rand((b, hkv, 1, d), dtype, 84, 40.0)
    slots = [int(table[i, (n - 1) // page]) * page + (n - 1) % page if n else -1 for i, n in enumerate(lens)]
    slots[4] = slots[7] = -1                     # no new row: they attend to what they have
    nv[3, 0, 0, 2] = math.nan                    # not finite: its row stands for NaN
    slots = torch.tensor(slots, device="cuda")
    # a request of no new row sees a row there
    mine, other = [x.clone() for x in cache], [x.clone() for x in cache]
    if d % 16:
        mine = [_like(x) for x in cache[:2]] + mine[2:]
        other = [_like(x) for x in cache[:2]] + other[2:]
    out, lse = paged_attention8(q, *mine, table, lengths, new_k=nk, new_v=nv, slots=slots, return_lse=True)
    append_paged_kv8(*other, nk, nv, slots)
    want, want_lse = paged_attention8(q, *other, table, lengths, return_lse=True)
    for x, y in zip(mine, other):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    g = hq // hkv
    assert torch.isnan(out[3, :g]).all() and torch.isfinite(lse[3]).all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[3, :g] = False
    assert torch.equal(out[keep], want[keep]) and torch.equal(lse, want_lse)
    assert torch.isfinite(out[keep]).all()


def _like(pages):
    """A copy with the same strides."""
    n, h, p, d = pages.shape
    wide = torch.zeros(n, h, p, pages.stride(2), device="cuda", dtype=torch.uint8).view(pages.dtype)[..., :d]
    wide.copy_(pages)
    return wide


# ---------------------------------------------------------------- all of it

@pytest.mark.parametrize("held,block,dtype", [(torch.float8_e4m3fn, 1, BF16), (torch.int8, 1, F16), (torch.int8, 16, BF16)])
def test_serving_with_rotary_positions(held, block, dtype):
    """Prompts, then a captured generation step, as a server runs them: rotate,
    reserve, append, attend; against the oracle over what the cache holds, which
    is what was stored, to a code's rounding."""
    hq, hkv, d, page, slots_n = 8, 2, 72, 16, 3
    cache = PagedKVCache8(40, page, hkv, d, slots_n, 10, layers=2, scale_block=block, device="cuda", dtype=held)
    freqs, magnitude = rotary_frequencies(64, scaling="yarn", factor=4.0, trained_length=32, device="cuda")
    prompts = [37, 5, 64]
    keys = [[[] for _ in range(slots_n)] for _ in range(2)]
    total = sum(prompts)
    added = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    rows, starts = cache.reserve(added, num_tokens=total)
    positions = torch.cat([torch.arange(n) for n in prompts]).to(torch.int32).cuda()[None]
    for layer in range(2):
        q, k, v = (_rand((1, total, h, d), dtype, 90 + layer * 3 + i).transpose(1, 2) for i, h in enumerate((hq, hkv, hkv)))
        _, k = apply_rotary(q, k, positions, freqs, magnitude=magnitude)
        cache.append(k, v, rows, layer=layer)
        back = cache.read(rows, dtype=dtype, layer=layer)
        for got, x in zip(back, (k, v)):
            top = x.abs().amax((-1, -2) if block > 1 else -1, keepdim=True).double()
            assert ((got.double() - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, top * 2.0 ** -7)).all()
    q, k, v = (_rand((slots_n, h, 1, d), dtype, 99 + i) for i, h in enumerate((hq, hkv, hkv)))
    active = torch.ones(slots_n, dtype=torch.int32, device="cuda")
    outs = [torch.empty_like(q) for _ in range(2)]

    def step():
        new, _ = cache.reserve(active, tokens_per_request=1)
        at = (cache.lengths - 1)[:, None]
        for layer in range(2):
            rq, rk = apply_rotary(q, k, at, freqs, magnitude=magnitude)
            outs[layer].copy_(cache.append_and_attend(rq, rk, v, new, layer=layer))
        return rq

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(side):
        held_rows = step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held_rows = step()
    torch.cuda.synchronize()
    for i in range(20):
        g = torch.Generator(device="cuda").manual_seed(500 + i)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda") * 3 ** (i % 3))
        if i == 11:
            active[1] = 0
        graph.replay()
    torch.cuda.synchronize()
    lens = [n + 21 for n in prompts]
    lens[1] = prompts[1] + 12
    assert cache.lengths.tolist() == lens
    for layer in range(2):
        kv, vv = (oracle8.values(getattr(cache, x)[layer].cpu().double(), oracle8.exps_of(getattr(cache, x + "_scales")[layer])) for x in "kv")
        _check(outs[layer], None, held_rows, kv, vv, cache.block_table, cache.lengths, d ** -0.5, f"layer {layer}")
    cache.release(torch.ones(slots_n, dtype=torch.bool, device="cuda"))
    assert int(cache.free_count) == 40
    del graph


def test_pools_past_4_gb():
    """Pages, rows and scales whose offsets need more than 32 bits: stored, read
    and attended to at both ends of a pool of 5 GB, as in a small one."""
    hkv, page, d, far = 8, 64, 128, 81000
    slots_at = lambda first: torch.arange(100, device="cuda") + first * page  # noqa: E731
    k, v, q = (_rand((1, 100, h, d), BF16, 96 + i).transpose(1, 2) for i, h in enumerate((hkv, hkv, 16)))
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([100], dtype=torch.int32, device="cuda")
    outs = []
    for pages, first in ((2, 0), (far + 2, far)):
        pools = [torch.empty(pages, hkv, page, d, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.empty(pages, hkv, page, device="cuda", dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2)]
        cache = (*pools, *scales)
        append_paged_kv8(*cache, k, v, slots_at(first))
        back = read_paged_kv8(*cache, slots_at(first), dtype=BF16)
        new = [x[:, :, 50:51].contiguous() for x in (k, v)]
        out = paged_attention8(q[:, :, :1].contiguous(), *cache, table + first, lengths, new_k=new[0], new_v=new[1],
                               slots=slots_at(first)[99:], return_lse=True)
        outs.append((*back, *out, *read_paged_kv8(*cache, slots_at(first)[99:], dtype=BF16)))
        del pools, scales, cache
    for x, y in zip(*outs):
        assert torch.equal(x, y)


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two CUDA devices")
def test_calls_follow_their_tensors_device():
    """Everything on cuda:1 while cuda:0 is current: the results of cuda:0."""
    results = []
    for index in (0, 1):
        dev = torch.device("cuda", index)
        with torch.cuda.device(index):
            g = torch.Generator(device=dev).manual_seed(1)
            q, k, v = (torch.randn(1, h, 40, 64, device=dev, generator=g).bfloat16() for h in (4, 2, 2))
            cache = PagedKVCache8(8, 16, 2, 64, 1, 4, device=dev)
            freqs, _ = rotary_frequencies(64, device=dev)
            torch.cuda.synchronize(dev)
        with torch.cuda.device(0):
            q, k = apply_rotary(q, k, torch.arange(40, device=dev), freqs)
            slots, _ = cache.reserve(torch.tensor([40], dtype=torch.int32, device=dev), num_tokens=40)
            cache.append(k, v, slots)
            out, lse = cache.attend(q[:, :, :1].contiguous(), return_lse=True)
            results.append([x.cpu() for x in (out, lse, *cache.read(slots, dtype=torch.float16))])
    for x, y in zip(*results):
        assert torch.equal(x, y)


def test_two_streams_at_once():
    """Two calls in flight with workspaces of their own."""
    cache, kv, vv, table, lengths = _requests([9000, 8000], 16, 2, 128, "e4m3", 91)
    q = [_rand((2, 8, 1, 128), BF16, 92 + i) for i in range(2)]
    want = [paged_attention8(x, *cache, table, lengths) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention8(q[i], *cache, table, lengths))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_nothing_to_do():
    cache, *_ , table, lengths = _requests([20], 16, 2, 64, "e4m3", 95)
    before = [x.view(torch.uint8).clone() for x in cache]
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    rows = torch.empty(1, 2, 0, 64, dtype=BF16, device="cuda")
    append_paged_kv8(*cache, rows, rows, none)
    k, v = read_paged_kv8(*cache, none, dtype=F16)
    assert k.shape == v.shape == (1, 2, 0, 64)
    out, lse = paged_attention8(_rand((1, 4, 1, 64), F16, 1), *cache, table, torch.zeros_like(lengths), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert all(torch.equal(x, y.view(torch.uint8)) for x, y in zip(before, cache))
