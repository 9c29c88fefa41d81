# SPDX-License-Identifier: Apache-2.0
"""The paged KV cache at its edges (GPU)."""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kotflash_b200 import PagedKVCache, append_paged_kv, paged_attention, reserve_pages
from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


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


# ---------------------------------------------------------------- infinities

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 2, 64, 16), (16, 1, 128, 16), (24, 1, 72, 24), (40, 1, 104, 8), (3, 3, 16, 5)])
def test_infinite_values_stay_infinite(dtype, hq, hkv, d, page):
    """O = sum w v with w > 0: +inf or -inf where a column sees one, NaN where
    it sees both or a NaN; every other column as without them."""
    lens = [100, 1, 33, 700, 9000, 60]
    g = torch.Generator(device="cuda").manual_seed(hq + d)
    held = [-(-n // page) for n in lens]
    cols = max(held)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = torch.arange(at, at + h)
        at += h
    shape = (at, hkv, page, d)
    k = torch.randn(shape, device="cuda", generator=g).to(dtype)
    v = torch.randn(shape, device="cuda", generator=g).to(dtype)
    q = (torch.randn(len(lens), hq, 1, d, device="cuda", generator=g) * 1.5).to(dtype)
    for b, n in enumerate(lens):                       # position, head, column, value
        for i in range(6 if n > 40 else 1):
            p = (i * 37 + b) % n
            v[int(table[b, p // page]), i % hkv, p % page, (5 * i + b) % d] = (math.inf, -math.inf, math.inf)[i % 3]
        if n > 40:                                     # a column with both, and one with a NaN
            for p, x in ((3, math.inf), (n - 2, -math.inf)):
                v[int(table[b, p // page]), 0, p % page, d - 1] = x
            v[int(table[b, 7 // page]), 0, 7 % page, d - 2] = math.nan
    table, lengths, scale = table.cuda(), _i32(lens), d ** -0.5
    out, lse = paged_attention(q, k, v, table, lengths, return_lse=True)
    want, want_lse, _ = oracle.attention(q, k, v, table, lengths, scale)
    finite = torch.isfinite(want)
    assert (~finite).any() and torch.isinf(want).any() and torch.isnan(want).any()
    got = out.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    tame = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    same, _, sizes = oracle.attention(q, k, tame, table, lengths, scale)
    for b, (prod, vmax, n) in enumerate(sizes):        # as for finite values: see the checks of ragged batches
        dx = prod * (d + 2) * 2.0 ** -23 + 2.0 ** -22
        bound = UNIT[dtype] * same[b].abs() + vmax * (2.0 ** -16 + 2 * dx + (n / 16 + 64) * 2.0 ** -23) + 2.0 ** -24
        off = torch.where(finite[b], (got[b] - same[b]).abs() - bound, -1.0)
        assert (off <= 0).all()
    assert torch.isfinite(lse).all()


def test_an_infinite_value_behind_a_small_weight():
    """fp16 holds a weight of 2^-40 of the largest as no number; its V still decides the sign of an infinity."""
    k = torch.zeros(4, 1, 16, 64, device="cuda", dtype=torch.float16)
    v = torch.ones_like(k)
    k[0, 0, 0, 0], v[3, 0, 2, 7], v[1, 0, 3, 9] = 40.0, math.inf, -math.inf
    q = torch.zeros(1, 1, 1, 64, device="cuda", dtype=torch.float16)
    q[..., 0] = 1
    out = paged_attention(q, k, v, _i32([[0, 1, 2, 3]]), _i32([64]), scale=math.log(2))[0, 0, 0]
    assert out[7] == math.inf and out[9] == -math.inf
    assert (out[[c for c in range(64) if c not in (7, 9)]] == 1).all()


def test_a_scale_of_zero_leaves_no_score():
    """Products of 1e38 included: all weights are equal."""
    k = torch.full((4, 1, 16, 64), 0.0, device="cuda", dtype=torch.bfloat16)
    k[:, :, ::2, 0], k[:, :, 1::2, 0] = 1e19, -1e19
    v = torch.arange(64, device="cuda", dtype=torch.bfloat16)[:, None].expand(64, 64).reshape(4, 1, 16, 64).contiguous()
    q = torch.zeros(1, 1, 1, 64, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1e19
    for scale in (0.0, -0.0, 1e-60):
        out, lse = paged_attention(q, k, v, _i32([[0, 1, 2, 3]]), _i32([64]), scale=scale, return_lse=True)
        assert (out == 31.5).all() and abs(lse.item() - math.log(64)) < 4e-6


# ---------------------------------------------------------------- sizes of the tables

def _fresh(code, *args):
    """Runs code in a process of its own, where nothing of the package has been called yet."""
    done = subprocess.run([sys.executable, "-c", code, *map(str, args)], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout + done.stderr


def test_table_sizes_around_the_shared_memory_limit():
    """Batches whose tables of 12 (reserve) or 4 (release) bytes per request lie
    around 48 KB, from the smallest up, and the largest."""
    _fresh("""
import torch
from kotflash_b200 import release_pages, reserve_pages
i32 = dict(dtype=torch.int32, device="cuda")
for b in (4051, 4052, 4095, 4096, 16384):
    table = torch.full((b, 1), -1, **i32)
    slots, starts, lengths, count = reserve_pages(torch.zeros(b, **i32), torch.ones(b, **i32), table, torch.arange(b, **i32),
                                                  torch.full((1,), b, **i32), page_size=16, num_tokens=b)
    pages = torch.arange(b - 1, -1, -1, device="cuda")
    assert torch.equal(slots, pages * 16) and torch.equal(table[:, 0], pages.int()), b
    assert torch.equal(starts, torch.arange(b + 1, **i32)) and (lengths == 1).all() and count.item() == 0, b
for b in (12160, 12161, 12288, 12289, 16384):
    free = torch.full((b,), -1, **i32)
    lengths, count = release_pages(torch.ones(b, **i32), torch.ones(b, dtype=torch.bool, device="cuda"),
                                   torch.arange(b, **i32)[:, None], free, torch.zeros(1, **i32), page_size=16)
    assert torch.equal(free, torch.arange(b, **i32)) and (lengths == 0).all() and count.item() == b, b
""")


def test_reserve_gives_no_token_without_a_slot():
    """Packed slots that end before a request's tokens do: the request is refused, and so are those after it."""
    def reserve(added, num_tokens):
        b = len(added)
        table = torch.full((b, 4), -1, dtype=torch.int32, device="cuda")
        free = torch.arange(10, dtype=torch.int32, device="cuda")
        slots, starts, lengths, count = reserve_pages(_i32([0] * b), _i32(added), table, free, _i32([10]), page_size=4,
                                                      num_tokens=num_tokens)
        return slots.tolist(), starts.tolist(), lengths.tolist(), count.item(), table.tolist()

    slots, starts, lengths, count, table = reserve([3, 5, 0, 2, 0], 9)
    assert slots == [36, 37, 38, 32, 33, 34, 35, 28, -1] and starts == [0, 3, 8, 8, 10, 10]
    assert lengths == [3, 5, 0, 0, 0] and count == 7
    assert table == [[9, -1, -1, -1], [8, 7, -1, -1]] + [[-1] * 4] * 3
    assert reserve([3, 5, 0, 2, 0], 8)[2] == [3, 5, 0, 0, 0]
    assert reserve([3, 5, 0, 2, 0], 7)[2] == [3, 0, 0, 0, 0]
    assert reserve([3, 5, 0, 2, 0], 10)[2] == [3, 5, 0, 2, 0]
    assert reserve([3, 1], 0) == ([], [0, 3, 4], [0, 0], 10, [[-1] * 4] * 2)


# ---------------------------------------------------------------- nothing to store

def test_appending_no_tokens():
    """A step that admits no prompt: no slots, no rows, nothing stored."""
    cache = PagedKVCache(6, 16, 2, 64, 3, 2, device="cuda", dtype=torch.float16)
    cache.k.zero_()
    cache.v.zero_()
    slots, starts = cache.reserve(_i32([0, 0, 0]), num_tokens=0)
    assert slots.shape == (0,) and starts.tolist() == [0, 0, 0, 0]
    rows = torch.ones(1, 2, 0, 64, device="cuda", dtype=torch.float16)
    cache.append(rows, rows, slots)
    none = torch.ones(0, 2, 5, 64, device="cuda", dtype=torch.float16)
    append_paged_kv(cache.k[0], cache.v[0], none, none, slots)
    assert not cache.k.any() and not cache.v.any()
    for k, v, match in ((rows[:, :1], rows[:, :1], "heads"), (rows[..., :32], rows[..., :32], "head"), (rows, none, "shapes")):
        with pytest.raises(ValueError, match=match):
            cache.append(k, v, slots)


# ---------------------------------------------------------------- the first call of a process

def test_first_reserve_under_a_tracing_mode():
    """A call on tensors without memory fails; the process's later calls do not."""
    _fresh("""
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from kotflash_b200 import reserve_pages
i32 = dict(dtype=torch.int32, device="cuda")
def reserve():
    return reserve_pages(torch.zeros(2, **i32), torch.ones(2, **i32), torch.full((2, 4), -1, **i32), torch.arange(9, **i32),
                         torch.full((1,), 9, **i32), page_size=16, num_tokens=2)
try:
    with FakeTensorMode():
        reserve()
except Exception as exc:
    print(type(exc), exc)
else:
    raise SystemExit("a call without memory went through")
assert reserve()[0].tolist() == [128, 112]
""")


_FIRST = """
import torch
from kotflash_b200 import _ext, paged_attention
dev = torch.device("cuda", 0)
def attend():
    f16, i32 = dict(dtype=torch.float16, device="cuda"), dict(dtype=torch.int32, device="cuda")
    return paged_attention(torch.zeros(1, 2, 1, 64, **f16), torch.zeros(4, 2, 16, 64, **f16), torch.zeros(4, 2, 16, 64, **f16),
                           torch.zeros(1, 4, **i32), torch.full((1,), 40, **i32))
"""


def test_first_call_in_inference_mode():
    _fresh(_FIRST + """
with torch.inference_mode():
    attend()
_ext.clear_device_status(dev)
assert _ext.read_device_status(dev) == 0
""")


def test_first_call_inside_a_graph_capture():
    """The status word is not cleared by the graph's replays."""
    _fresh(_FIRST + """
f16, i32 = dict(dtype=torch.float16, device="cuda"), dict(dtype=torch.int32, device="cuda")
q, k = torch.zeros(1, 2, 1, 64, **f16), torch.zeros(4, 2, 16, 64, **f16)
table, lengths = torch.zeros(1, 4, **i32), torch.full((1,), 40, **i32)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = paged_attention(q, k, k, table, lengths)
word = _ext.status_word(dev)
assert word.item() == 0 and _ext.read_device_status(dev) == 0
word.fill_(1)
graph.replay()
torch.cuda.synchronize()
assert _ext.read_device_status(dev) == 1
_ext.clear_device_status(dev)
assert _ext.read_device_status(dev) == 0 and (out == 0).all()
del graph
""")


def test_first_attention_under_a_tracing_mode():
    """A call on tensors without memory fails; the status word of later calls is there."""
    _fresh(_FIRST + """
from torch._subclasses.fake_tensor import FakeTensorMode
try:
    with FakeTensorMode():
        attend()
except Exception as exc:
    print(type(exc), exc)
else:
    raise SystemExit("a call without memory went through")
assert (attend() == 0).all()
_ext.status_word(dev).fill_(1)
assert _ext.read_device_status(dev) == 1
_ext.clear_device_status(dev)
assert _ext.read_device_status(dev) == 0
""")
