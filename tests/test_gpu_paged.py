# SPDX-License-Identifier: Apache-2.0
"""K5/K6, the paged KV cache, against the 64-bit oracle (GPU)."""
import math

import pytest
import torch

from kotflash_b200 import PagedKVCache, append_paged_kv, attention, paged_attention, release_pages, reserve_pages
from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # unit roundoff of the output's type


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def _pool(lens, page, hkv, d, dtype, seed, extra_cols=1, spare=3, fill=float("nan")):
    """A pool whose pages are handed out at random; every row that no request
    owns, and every table entry past a request's pages, is filled with junk."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lens]
    n_pages = sum(held) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    cols = max(held) + extra_cols
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    k = torch.full((n_pages, hkv, page, d), fill, device="cuda", dtype=dtype)
    v = torch.full((n_pages, hkv, page, d), fill, device="cuda", dtype=dtype)
    src_k = _rand((n_pages, hkv, page, d), dtype, seed + 1)
    src_v = _rand((n_pages, hkv, page, d), dtype, seed + 2)
    at = 0
    for b, n in enumerate(lens):
        for j in range(held[b]):
            p = order[at]
            at += 1
            table[b, j] = p
            rows = min(page, n - j * page)
            k[p, :, :rows] = src_k[p, :, :rows]
            v[p, :, :rows] = src_v[p, :, :rows]
        # entries past the end name real pages and nonsense in turn
        for j in range(held[b], cols):
            table[b, j] = order[j % n_pages] if j % 2 else -1 if j % 4 else 2**31 - 1
    return k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def _check(out, lse, q, k, v, table, lengths, scale, name):
    """Bounds: a score is a sum of D products in fp32 (error at most D 2^-23
    sum |q_i k_i| scale, tensor cores truncating) and enters a weight through a
    base-2 exponential (argument rounding |x| 2^-23, function 2^-22); the
    weights are held as two 16-bit parts (2^-16 together in bf16, the coarser
    type); products and weights are summed 16 at a time in fp32 over n keys,
    plus a handful of joins; the output is rounded once (unit roundoff u)."""
    eo, el, sizes = oracle.attention(q, k, v, table, lengths, scale)
    o = out.double().cpu()
    d = q.shape[-1]
    assert out.shape == q.shape and out.dtype == q.dtype
    for b, (prod, vmax, n) in enumerate(sizes):
        if n == 0:
            assert (o[b] == 0).all(), f"{name}: request {b} sees nothing"
            assert lse is None or (lse[b] == -math.inf).all()
            continue
        dx = prod * (d + 2) * 2.0 ** -23 + 2.0 ** -22
        weight = 2.0 ** -16 + 2 * dx + (n / 16 + 64) * 2.0 ** -23
        err = (o[b] - eo[b]).abs()
        bound = UNIT[q.dtype] * eo[b].abs() + vmax * weight + 2.0 ** -24
        assert (err <= bound).all(), f"{name}: request {b} (n={n}) off by {err.max():.3e}, bound {bound.min():.3e}"
        if lse is not None:
            assert lse.shape == q.shape[:3] and lse.dtype == torch.float32
            el_b = (lse[b].double().cpu() - el[b]).abs().max().item()
            assert el_b <= dx + (n / 16 + 64) * 2.0 ** -23 + el[b].abs().max().item() * 2.0 ** -22, f"{name}: LSE {b} off by {el_b}"


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1999]


@pytest.mark.parametrize("hq,hkv,d,dtype,page", [
    (8, 2, 64, torch.float16, 16),
    (32, 8, 128, torch.bfloat16, 16),
    (4, 4, 128, torch.float16, 64),      # one row per KV head
    (6, 2, 72, torch.bfloat16, 24),      # pages that end inside a tile
    (8, 1, 104, torch.float16, 5),
    (12, 1, 128, torch.bfloat16, 1),     # two row tiles, one position per page
    (16, 1, 64, torch.float16, 3),
    (24, 1, 128, torch.float16, 100),    # a team of two warps
    (32, 1, 40, torch.bfloat16, 8),
    (40, 1, 128, torch.bfloat16, 32),    # a team of four
    (64, 1, 16, torch.float16, 256),
    (72, 1, 96, torch.bfloat16, 16),     # two row blocks
    (130, 2, 24, torch.float16, 7),
])
def test_ragged_batches_against_the_oracle(hq, hkv, d, dtype, page):
    k, v, table, lengths = _pool(LENS, page, hkv, d, dtype, 11)
    q = _rand((len(LENS), hq, 1, d), dtype, 7, 1.5)
    out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    _check(out, lse, q, k, v, table, lengths, d ** -0.5, f"{hq},{hkv},{d},{page}")
    again = paged_attention(q, k, v, table, lengths)
    assert torch.equal(out, again)  # the same sums in the same order, with and without the LSE


@pytest.mark.parametrize("d", range(16, 129, 8))
@pytest.mark.parametrize("page", [4, 8, 16, 32])
def test_every_head_dim_and_tile_layout(d, page):
    """Every way a tile lies in shared memory: panels of 64, 32 and 16 columns,
    dense rows, boxes of 4 to 32 rows, both team shapes."""
    lens = [33, 1, 150, 260]
    for hq, dtype in ((6, torch.bfloat16), (40, torch.float16)):
        k, v, table, lengths = _pool(lens, page, 2, d, dtype, 200 + d + page)
        q = _rand((len(lens), hq, 1, d), dtype, 201, 1.5)
        out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
        _check(out, lse, q, k, v, table, lengths, d ** -0.5, f"layout {d},{page},{hq}")


@pytest.mark.parametrize("hq,hkv,d,dtype,page,lens", [
    (8, 2, 64, torch.float16, 64, [30000, 12345]),         # few requests: many partials to join
    (4, 1, 128, torch.bfloat16, 16, [20011]),
    (32, 1, 128, torch.float16, 16, [5000, 1]),
    (64, 1, 64, torch.bfloat16, 32, [9000]),
    (8, 8, 128, torch.bfloat16, 16, [1] * 100 + [700] * 50 + [0] * 200 + [33] * 200),  # more requests than threads
])
def test_long_and_many(hq, hkv, d, dtype, page, lens):
    k, v, table, lengths = _pool(lens, page, hkv, d, dtype, 21)
    q = _rand((len(lens), hq, 1, d), dtype, 8)
    out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    _check(out, lse, q, k, v, table, lengths, d ** -0.5, f"long {hq},{hkv},{d},{page}")


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 8, 1), (128, 24, 1), (64, 64, 1)])
def test_every_position_counts_once(d, hq, hkv):
    """With q = 0 all weights are equal: LSE = ln(number of visible positions),
    to 64-bit-against-fp32 accuracy, and O is the mean of small whole numbers."""
    lens = list(range(0, 140)) + [1000, 4097, 10000]
    k, v, table, lengths = _pool(lens, 16, hkv, d, torch.bfloat16, 31)
    junk = torch.isnan(v)
    v = (torch.arange(v.numel(), device="cuda") % 7 - 3).view(v.shape).to(v.dtype)
    v[junk] = float("nan")
    q = torch.zeros(len(lens), hq, 1, d, device="cuda", dtype=torch.bfloat16)
    out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    _check(out, None, q, k, v, table, lengths, d ** -0.5, "mean")
    want = torch.log(torch.tensor(lens, dtype=torch.float64))
    # one position of 10000 moves the LSE by 1e-4; fp32 holds 9.2 to 1e-6
    got = lse.double().cpu()[..., 0]
    assert ((got - want[:, None]).abs()[1:] < 4e-6).all() and (got[0] == -math.inf).all()


def test_layouts_and_strides():
    """Pages with tokens outside heads, K and V with different strides, q and
    the table as slices of larger tensors."""
    lens, hq, hkv, d, page = [70, 0, 333, 16], 8, 2, 64, 16
    k, v, table, lengths = _pool(lens, page, hkv, d, torch.float16, 41)
    q = _rand((4, hq, 1, d), torch.float16, 42)
    want, want_lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    k2 = k.transpose(1, 2).contiguous().transpose(1, 2)              # [pages, page, Hkv, D] in memory
    pair = torch.empty(k.shape[0], 2, hkv, page, d + 8, device="cuda", dtype=k.dtype)
    v2 = pair[:, 1, :, :, :d]
    v2.copy_(v)
    fused = torch.empty(4, (hq + 2 * hkv) * d, device="cuda", dtype=q.dtype)
    q2 = fused[:, : hq * d].view(4, hq, 1, d)
    q2.copy_(q)
    wide = torch.full((4, table.shape[1] + 5), -7, device="cuda", dtype=torch.int32)
    wide[:, : table.shape[1]] = table
    got, got_lse = paged_attention(q2, k2, v2, wide[:, : table.shape[1]], lengths, return_lse=True)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    # the same requests in another order, and each alone, where its shares differ
    back = torch.tensor([3, 2, 1, 0], device="cuda")
    assert torch.equal(paged_attention(q[back], k, v, table[back], lengths[back])[back][1], want[1])
    for b in range(4):
        one, one_lse = paged_attention(q[b:b + 1], k, v, table[b:b + 1], lengths[b:b + 1], return_lse=True)
        _check(one, one_lse, q[b:b + 1], k, v, table[b:b + 1], lengths[b:b + 1], d ** -0.5, f"alone {b}")


def test_masked_positions_are_not_read():
    """Table entries outside the pool mask their positions; lengths below 0
    count as 0 and above the table's room as full; NaN fills all of it."""
    lens, hq, hkv, d, page = [160, 160, 160, 40, 40], 4, 2, 64, 16
    k, v, table, lengths = _pool(lens, page, hkv, d, torch.bfloat16, 51, extra_cols=0)
    table[0, 3] = -1
    table[1, :] = k.shape[0]              # no position left
    table[2, 0], table[2, 9] = -2**31, 2**31 - 1
    lengths[3] = -5
    lengths[4] = 2**31 - 1                # the table ends at 160
    table[4, 3:] = table[4, :1]           # ... with entries that are pages
    q = _rand((5, hq, 1, d), torch.bfloat16, 52)
    k[table[4, 2], :, 8:] = 0.5
    v[table[4, 2], :, 8:] = 0.25
    out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    assert torch.isfinite(out).all()
    _check(out, lse, q, k, v, table, lengths, d ** -0.5, "masked")


def test_nan_and_infinity_stay_in_their_request():
    lens, hq, hkv, d, page = [100, 100, 100, 2000], 4, 2, 128, 16
    k, v, table, lengths = _pool(lens, page, hkv, d, torch.bfloat16, 61)
    q = _rand((4, hq, 1, d), torch.bfloat16, 62)
    want = paged_attention(q, k, v, table, lengths)
    k[table[0, 2], 0, 3, 5] = float("nan")
    v[table[1, 2], 1, 3, 5] = float("inf")
    out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    assert torch.isnan(out[0, :2]).all() and torch.isnan(lse[0, :2]).all()
    assert torch.equal(out[0, 2:], want[0, 2:])
    assert not torch.isfinite(out[1, 2:, 0, 5]).any() and torch.isfinite(lse[1]).all()
    others = [c for c in range(d) if c != 5]
    assert torch.equal(out[1][..., others], want[1][..., others]) and torch.equal(out[1, :2], want[1, :2])
    assert torch.equal(out[2:], want[2:])


def test_large_scores_and_scales():
    lens, hq, hkv, d, page = [300, 17], 4, 2, 64, 16
    k, v, table, lengths = _pool(lens, page, hkv, d, torch.bfloat16, 71)
    q = _rand((2, hq, 1, d), torch.bfloat16, 72, 40.0)
    for scale in (1.0, -0.5, 0.0, 1e-4):
        out, lse = paged_attention(q, k, v, table, lengths, scale=scale, return_lse=True)
        _check(out, lse, q, k, v, table, lengths, scale, f"scale {scale}")


def test_offsets_past_32_bits():
    """A pool of 2^31 + elements per tensor, the request's pages at its far end."""
    hkv, page, d = 8, 256, 128
    n_pages = (2**31) // (hkv * page * d) + 40
    k = torch.empty(n_pages, hkv, page, d, device="cuda", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    table = torch.tensor([[n_pages - 1, 0, n_pages - 7], [n_pages - 20, n_pages - 30, -1]], dtype=torch.int32, device="cuda")
    for p in (n_pages - 1, 0, n_pages - 7, n_pages - 20, n_pages - 30):
        k[p] = _rand((hkv, page, d), torch.bfloat16, p % 1000)
        v[p] = _rand((hkv, page, d), torch.bfloat16, p % 1000 + 1)
    lengths = torch.tensor([700, 512], dtype=torch.int32, device="cuda")
    q = _rand((2, 16, 1, d), torch.bfloat16, 82)
    nk, nv = _rand((2, hkv, 1, d), torch.bfloat16, 83), _rand((2, hkv, 1, d), torch.bfloat16, 84)
    last = torch.tensor([(n_pages - 7) * page + 699 - 512, (n_pages - 30) * page + 255], device="cuda")
    append_paged_kv(k, v, nk, nv, last)
    assert torch.equal(k[n_pages - 7, :, 699 - 512], nk[0, :, 0]) and torch.equal(v[n_pages - 30, :, 255], nv[1, :, 0])
    out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    _check(out, lse, q, k, v, table, lengths, d ** -0.5, "far pages")


@pytest.mark.parametrize("seed", range(40))
def test_random_cases(seed):
    """Seeded draws over heads, head dims, pages, lengths, layouts, masked table
    entries and the fused append, which must equal appending first."""
    import random

    r = random.Random(seed)
    hkv = r.choice([1, 2, 3, 5, 8])
    hq = hkv * r.choice([1, 2, 3, 4, 7, 8, 9, 16, 17, 33, 65][: 11 if hkv < 3 else 6])
    d = 8 * r.randint(2, 16)
    page = r.choice([1, 2, 3, 8, 12, 16, 16, 32, 40, 64, 128])
    dtype = r.choice([torch.float16, torch.bfloat16])
    top = r.choice([3, 40, 200, 1500])
    lens = [r.choice([0, 1, top, r.randint(0, top), r.randint(0, top)]) for _ in range(r.choice([1, 2, 7, 40, 130]))]
    if not any(lens):
        lens[0] = top
    k, v, table, lengths = _pool(lens, page, hkv, d, dtype, 1000 + seed)
    if r.random() < 0.5:  # tokens outside heads
        k = k.transpose(1, 2).contiguous().transpose(1, 2)
    for b, n in enumerate(lens):  # some pages in the middle are given up
        held = -(-n // page)
        if held > 1 and r.random() < 0.3:
            table[b, r.randrange(held - 1)] = r.choice([-1, k.shape[0], -2**31])
    q = _rand((len(lens), hq, 1, d), dtype, 2000 + seed, r.choice([0.5, 2.0]))
    scale = r.choice([None, None, 0.3, -0.1])
    out, lse = paged_attention(q, k, v, table, lengths, scale=scale, return_lse=True)
    _check(out, lse, q, k, v, table, lengths, d ** -0.5 if scale is None else scale, f"seed {seed}")
    nk, nv = _rand((len(lens), hkv, 1, d), dtype, 3000 + seed), _rand((len(lens), hkv, 1, d), dtype, 4000 + seed)
    slots = torch.tensor([int(table[b, (n - 1) // page]) * page + (n - 1) % page if n and r.random() < 0.8 else -1
                          for b, n in enumerate(lens)], device="cuda")
    k2, v2 = k.clone(), v.clone()
    got = paged_attention(q, k2, v2, table, lengths, scale=scale, new_k=nk, new_v=nv, slots=slots)
    append_paged_kv(k, v, nk, nv, slots)
    assert torch.equal(got, paged_attention(q, k, v, table, lengths, scale=scale))
    assert torch.equal(k.view(torch.int16), k2.view(torch.int16)) and torch.equal(v.view(torch.int16), v2.view(torch.int16))


# ---------------------------------------------------------------- fused append

@pytest.mark.parametrize("hq,hkv,d,dtype,page", [
    (8, 2, 64, torch.float16, 16), (32, 8, 128, torch.bfloat16, 16), (16, 1, 72, torch.bfloat16, 24),
    (32, 1, 96, torch.float16, 1), (72, 1, 128, torch.bfloat16, 32)])
def test_fused_append_equals_append_then_attend(hq, hkv, d, dtype, page):
    lens = [1, 2, 16, 17, 64, 65, 128, 700, 0, 31]
    k, v, table, lengths = _pool(lens, page, hkv, d, dtype, 91)
    q = _rand((len(lens), hq, 1, d), dtype, 92)
    both = _rand((2, hkv, len(lens), d), dtype, 93)   # rows with other strides than theirs alone
    nk, nv = both[0].transpose(0, 1)[:, :, None], both[1].transpose(0, 1)[:, :, None]
    slots = torch.full((len(lens),), -1, dtype=torch.int64, device="cuda")
    for b, n in enumerate(lens):
        if n and b != 4:                              # request 4 brings nothing this time
            slots[b] = int(table[b, (n - 1) // page]) * page + (n - 1) % page
    k1, v1, k2, v2 = k.clone(), v.clone(), k.clone(), v.clone()
    append_paged_kv(k1, v1, nk, nv, slots)
    want, want_lse = paged_attention(q, k1, v1, table, lengths, return_lse=True)
    got, got_lse = paged_attention(q, k2, v2, table, lengths, new_k=nk, new_v=nv, slots=slots, return_lse=True)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    bits = torch.int16                                # NaN junk compares by its bits
    assert torch.equal(k1.view(bits), k2.view(bits)) and torch.equal(v1.view(bits), v2.view(bits))
    assert not torch.equal(k2.view(bits), k.view(bits))


def test_fused_append_without_a_page_stores_nothing():
    k, v, table, lengths = _pool([20, 20], 16, 2, 64, torch.float16, 95)
    table[0, 1] = -1
    q = _rand((2, 4, 1, 64), torch.float16, 96)
    nk, nv = _rand((2, 2, 1, 64), torch.float16, 97), _rand((2, 2, 1, 64), torch.float16, 98)
    slots = torch.tensor([5, int(table[1, 1]) * 16 + 3], device="cuda")
    before_k = k.clone()
    out, lse = paged_attention(q, k, v, table, lengths, new_k=nk, new_v=nv, slots=slots, return_lse=True)
    _check(out, lse, q, k, v, table, lengths, 0.125, "no page")
    same = (k.view(torch.int16) == before_k.view(torch.int16)).all(-1)
    same[table[1, 1].long(), :, 3] = True
    assert same.all()


# ---------------------------------------------------------------- streams, graphs

def test_side_stream_and_graph_follow_the_lengths():
    lens, hq, hkv, d, page = [500, 3, 64], 8, 2, 64, 16
    k, v, table, lengths = _pool(lens, page, hkv, d, torch.float16, 101)
    q = _rand((3, hq, 1, d), torch.float16, 102)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = paged_attention(q, k, v, table, lengths)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, paged_attention(q, k, v, table, lengths))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    for now in ([500, 3, 64], [123, 0, 1], [1, 2, 33]):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        _check(out, lse, q, k, v, table, lengths, d ** -0.5, f"graph {now}")
    del g


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("n,s,hkv,d,page", [(1, 1, 1, 16, 1), (5, 1, 2, 64, 16), (1, 700, 8, 128, 16), (3, 33, 3, 72, 24),
                                            (1, 9000, 4, 64, 64), (2, 50, 33, 128, 8), (4, 7, 2, 20, 5), (1, 40, 1, 3, 4)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_is_bit_exact(n, s, hkv, d, page, dtype):
    t = n * s
    n_pages = -(-t // page) + 4
    g = torch.Generator().manual_seed(5)
    slots = torch.randperm(n_pages * page, generator=g)[:t].cuda()
    if t > 4:
        slots[1], slots[3] = -1, n_pages * page + 2   # neither is stored
    k, v = _rand((n_pages, hkv, page, d), dtype, 1), _rand((n_pages, hkv, page, d), dtype, 2)
    src = _rand((n, s, 2, hkv, d), dtype, 3)           # the projection's layout
    nk, nv = src[:, :, 0].transpose(1, 2), src[:, :, 1].transpose(1, 2)
    ek, ev = k.clone(), v.clone()
    rows_k, rows_v = nk.transpose(1, 2).reshape(t, hkv, d), nv.transpose(1, 2).reshape(t, hkv, d)
    ok = (slots >= 0) & (slots < n_pages * page)
    ek[slots[ok] // page, :, slots[ok] % page] = rows_k[ok]
    ev[slots[ok] // page, :, slots[ok] % page] = rows_v[ok]
    pools = torch.stack((k, v), 1)                     # K and V interleaved page by page
    append_paged_kv(pools[:, 0], pools[:, 1], nk, nv, slots)
    assert torch.equal(pools[:, 0], ek) and torch.equal(pools[:, 1], ev)
    hnd = k.transpose(1, 2).contiguous().transpose(1, 2)
    append_paged_kv(hnd, v, nk, nv, slots)
    assert torch.equal(hnd, ek) and torch.equal(v, ev)


# ---------------------------------------------------------------- tables

def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _table_case(b, page, high, seed, spare):
    import random

    r = random.Random(seed)
    lens = [r.choice([0, 1, page - 1, page, page + 1, r.randint(0, high)]) for _ in range(b)]
    held = [-(-n // page) for n in lens]
    num_pages = sum(held) + spare
    order = list(range(num_pages))
    r.shuffle(order)
    cols = -(-high // page) + 2
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-1] * (cols - h))
        at += h
    free = order[at:] + [-9] * at
    return r, lens, table, free, len(order) - at


@pytest.mark.parametrize("b,page,high,spare", [(1, 16, 50, 10), (7, 4, 90, 40), (33, 1, 20, 200), (300, 16, 700, 100), (1100, 8, 60, 900)])
@pytest.mark.parametrize("most", [1, 70])
@pytest.mark.parametrize("padded", [False, True])
def test_reserve_against_the_oracle(b, page, high, spare, most, padded):
    """Stacks that run out and rows that overflow included."""
    r, lens, table, free, count = _table_case(b, page, high, b + most, spare)
    added = [r.choice([0, 1, most, r.randint(0, most), -2]) for _ in range(b)]
    total = sum(max(x, 0) for x in added)
    kw = dict(tokens_per_request=max(1, most - 3)) if padded else dict(num_tokens=total + 5)
    want = oracle.reserve(lens, added, table, free, count, page, kw.get("num_tokens"), kw.get("tokens_per_request"))
    dt = _i32(table)
    dl, dc, df = _i32(lens), _i32([count]), _i32(free)
    slots, starts, out_l, out_c = reserve_pages(dl, _i32(added), dt, df, dc, page_size=page, **kw)
    assert slots.dtype == torch.int64 and slots.tolist() == want[0]
    assert starts.tolist() == want[1] and out_l.tolist() == want[2] and out_c.tolist() == [want[3]]
    assert dt.tolist() == want[4]
    assert dl.tolist() == lens and dc.tolist() == [count] and df.tolist() == free  # inputs stay
    # in place, and with a table that is a slice
    wide = torch.full((b, len(table[0]) + 3), -5, dtype=torch.int32, device="cuda")
    wide[:, : len(table[0])] = _i32(table)
    slots2, _, l2, c2 = reserve_pages(dl, _i32(added), wide[:, : len(table[0])], df, dc, page_size=page,
                                      lengths_out=dl, free_count_out=dc, **kw)
    assert torch.equal(slots, slots2) and l2 is dl and dl.tolist() == want[2] and dc.tolist() == [want[3]]
    assert wide[:, : len(table[0])].tolist() == want[4] and (wide[:, len(table[0]):] == -5).all()


def test_reserve_long_prompts_and_too_few_slots():
    """Token counts that need the whole cluster; fewer slots than tokens writes no further."""
    lens, added, page = [5, 0, 100, 0], [9000, 30001, 0, 4097], 16
    free = list(range(4000))
    table = [[-1] * 2000 for _ in lens]
    table[0][0], table[2][:7] = 3999, [3998 - i for i in range(7)]
    total = sum(added)
    for num in (total, total - 1001, 1, 0):
        want = oracle.reserve(lens, added, table, free, 3900, page, num)
        dt = _i32(table)
        slots, starts, out_l, out_c = reserve_pages(_i32(lens), _i32(added), dt, _i32(free), _i32([3900]), page_size=page, num_tokens=num)
        assert slots.tolist() == want[0] and starts.tolist() == want[1]
        assert out_l.tolist() == want[2] and out_c.tolist() == [want[3]] and dt.tolist() == want[4]


@pytest.mark.parametrize("b,page,high", [(1, 16, 50), (9, 4, 300), (40, 1, 20), (300, 16, 700), (1100, 8, 60)])
@pytest.mark.parametrize("every", [1, 3])
def test_release_against_the_oracle(b, page, high, every):
    r, lens, table, free, count = _table_case(b, page, high, b, 50)
    for row in table[::5]:                       # pages given up earlier
        if row[0] >= 0 and len(row) > 2:
            row[r.randrange(len(row) - 1)] = r.choice([-1, len(free), -2**31])
    finished = [i % every == 0 for i in range(b)]
    for cap in (count, 0, len(free) - 2, len(free) + 9):   # the last two overflow the stack
        want = oracle.release(lens, finished, table, free, cap, page)
        df = _i32(free)
        dl, dc = _i32(lens), _i32([cap])
        out_l, out_c = release_pages(dl, torch.tensor(finished, device="cuda"), _i32(table), df, dc, page_size=page)
        assert out_l.tolist() == want[0] and out_c.tolist() == [want[1]] and df.tolist() == want[2]
        assert dl.tolist() == lens and dc.tolist() == [cap]


def test_lifecycle_owns_every_page_once():
    """Random arrivals and departures: no page is ever owned twice, none is lost,
    and attention over what was written matches the oracle at the end."""
    import random

    r = random.Random(3)
    n_req, page, hkv, d, pages = 12, 4, 2, 64, 60
    cache = PagedKVCache(pages, page, hkv, d, n_req, 20, layers=2, device="cuda", dtype=torch.bfloat16)
    texts = [[] for _ in range(n_req)]           # seeds of the rows each request holds
    def row(seed):
        return _rand((2, 2, hkv, d), torch.bfloat16, seed)  # [layer, K or V]

    seed = 1000
    for step in range(25):
        added = [r.choice([0, 0, 1, 2, 5, 11]) if texts[b] else r.choice([0, 3, 17]) for b in range(n_req)]
        total = sum(added)
        before = cache.lengths.tolist()
        slots, starts = cache.reserve(_i32(added), num_tokens=total)
        after = cache.lengths.tolist()
        rows = [row(seed + i) for i in range(total)]
        for layer in range(2):
            if total:
                kv = torch.stack([x[layer] for x in rows], 1)   # [2, T, Hkv, D]
                cache.append(kv[0][None].transpose(1, 2), kv[1][None].transpose(1, 2), slots, layer=layer)
        for b in range(n_req):
            if after[b] > before[b]:
                assert after[b] - before[b] == added[b]
                texts[b] += list(range(seed + starts[b], seed + starts[b] + added[b]))
            else:
                assert (slots[starts[b]:starts[b] + added[b]] == -1).all()
        seed += total
        finished = [bool(texts[b]) and r.random() < 0.15 for b in range(n_req)]
        cache.release(torch.tensor(finished, device="cuda"))
        for b in range(n_req):
            if finished[b]:
                texts[b] = []
        lens, table = cache.lengths.tolist(), cache.block_table.tolist()
        assert lens == [len(t) for t in texts]
        owned = [p for b in range(n_req) for p in table[b][: -(-lens[b] // page)]]
        free = cache.free_pages[: int(cache.free_count)].tolist()
        assert sorted(owned + free) == list(range(pages))
    q = _rand((n_req, 4, 1, d), torch.bfloat16, 5)
    for layer in range(2):
        for b in range(n_req):
            for p, s in enumerate(texts[b]):
                assert torch.equal(cache.k[layer, cache.block_table[b, p // page], :, p % page], row(s)[layer, 0])
        out, lse = cache.attend(q, layer=layer, return_lse=True)
        _check(out, lse, q, cache.k[layer], cache.v[layer], cache.block_table, cache.lengths, 0.125, f"layer {layer}")


def test_pages_agree_with_the_contiguous_path():
    """The same keys through the pages and through attention() on a contiguous cache."""
    b, hq, hkv, n, d, page = 3, 8, 2, 777, 128, 16
    k, v = _rand((b, hkv, n, d), torch.bfloat16, 1), _rand((b, hkv, n, d), torch.bfloat16, 2)
    q = _rand((b, hq, 1, d), torch.bfloat16, 3)
    cache = PagedKVCache(200, page, hkv, d, b, 60, device="cuda", dtype=torch.bfloat16)
    slots, _ = cache.reserve(_i32([n] * b), tokens_per_request=n)
    cache.append(k, v, slots)
    with torch.no_grad():
        want = attention(q, k, v, backend="triton")
    torch.testing.assert_close(cache.attend(q).float(), want.float(), atol=2e-2, rtol=2e-2)
