# SPDX-License-Identifier: Apache-2.0
"""Paged KV cache on the CPU: refusals of the Python layer and of the C ABI
(before any launch), and the arithmetic of the decode kernel's work split."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import kotflash_b200 as kotflash
from kotflash_b200 import PagedKVCache, _ext, append_paged_kv, paged_attention, release_pages, reserve_pages
from oracle import paged_oracle as oracle


def _attend_args(**changes):
    a = dict(q=torch.zeros(3, 4, 1, 64, dtype=torch.float16), k_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float16),
             v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float16),
             block_table=torch.zeros(3, 2, dtype=torch.int32), lengths=torch.zeros(3, dtype=torch.int32))
    a.update(changes)
    return a


@pytest.mark.parametrize("changes,error,match", [
    (dict(q=None), TypeError, "torch.Tensor"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), TypeError, "lengths must be int32"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int64)), TypeError, "block_table must be int32"),
    (dict(block_table=[[0]]), TypeError, "block_table"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "block_table must be"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int32).t()), ValueError, "rows must be contiguous"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)), ValueError, "lengths must be"),
    (dict(lengths=torch.zeros(6, dtype=torch.int32)[::2]), ValueError, "lengths must be"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)), ValueError, "4-D"),
    (dict(q=torch.zeros(3, 4, 1, 64, dtype=torch.bfloat16)), ValueError, "dtypes must match"),
    (dict(q=torch.zeros(3, 5, 1, 64, dtype=torch.float16)), ValueError, "divisible"),
    (dict(q=torch.zeros(3, 0, 1, 64, dtype=torch.float16)), ValueError, "non-zero"),
    (dict(new_k=torch.zeros(3, 2, 1, 64, dtype=torch.float16)), ValueError, "go together"),
    (dict(slots=torch.zeros(3, dtype=torch.int64)), ValueError, "go together"),
    (dict(new_k=torch.zeros(3, 2, 1, 64, dtype=torch.float16), new_v=torch.zeros(3, 2, 1, 64, dtype=torch.float16),
          slots=torch.zeros(3, dtype=torch.int32)), TypeError, "slots must be int64"),
    (dict(new_k=torch.zeros(3, 2, 1, 64, dtype=torch.float16), new_v=torch.zeros(3, 2, 1, 64, dtype=torch.float16),
          slots=torch.zeros(2, dtype=torch.int64)), ValueError, "slots must be"),
    (dict(scale="x"), TypeError, "scale"),
    (dict(scale=float("inf")), ValueError, "finite"),
    (dict(q=torch.zeros(3, 4, 1, 64, dtype=torch.float16, requires_grad=True)), RuntimeError, "inference-only"),
    (dict(), RuntimeError, "sm_100"),
])
def test_paged_attention_refusals(changes, error, match):
    with pytest.raises(error, match=match):
        paged_attention(**_attend_args(**changes))


def test_paged_attention_needs_16_bit_tensors():
    a = {k: v.float() if v.is_floating_point() else v for k, v in _attend_args().items()}
    with pytest.raises(TypeError, match="float16 and bfloat16"):
        paged_attention(**a)


def test_append_refusals():
    pool = torch.zeros(5, 2, 16, 64, dtype=torch.float16)
    rows, slots = torch.zeros(1, 2, 3, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int64)
    for args, error, match in [
        ((pool, pool, rows, rows, slots.int()), TypeError, "int64"),
        ((pool, pool, rows, rows, slots[:2]), ValueError, "one slot for each"),
        ((pool, pool, rows, rows.bfloat16(), slots), ValueError, "dtypes"),
        ((pool, pool, rows[0], rows, slots), ValueError, "4-D"),
        ((pool, pool, rows, rows, None), TypeError, "torch.Tensor"),
        ((pool, pool, rows, rows, slots), RuntimeError, "sm_100"),
    ]:
        with pytest.raises(error, match=match):
            append_paged_kv(*args)


def test_table_refusals():
    i32 = torch.int32
    a = dict(lengths=torch.zeros(3, dtype=i32), new_lengths=torch.zeros(3, dtype=i32),
             block_table=torch.zeros(3, 2, dtype=i32), free_pages=torch.zeros(5, dtype=i32),
             free_count=torch.zeros(1, dtype=i32), page_size=16, num_tokens=0)
    for changes, error, match in [
        (dict(lengths=torch.zeros(3, dtype=torch.int64)), TypeError, "lengths must be int32"),
        (dict(new_lengths=torch.zeros(2, dtype=i32)), ValueError, "per-request"),
        (dict(block_table=torch.zeros(4, 2, dtype=i32)), ValueError, "block_table"),
        (dict(free_count=torch.zeros(2, dtype=i32)), ValueError, "free_count"),
        (dict(free_pages=torch.zeros(10, dtype=i32)[::2]), ValueError, "contiguous"),
        (dict(lengths_out=torch.zeros(2, dtype=i32)), ValueError, "lengths_out"),
        (dict(free_count_out=torch.zeros(1)), TypeError, "free_count_out"),
        (dict(), RuntimeError, "sm_100"),
    ]:
        with pytest.raises(error, match=match):
            reserve_pages(**{**a, **changes})
    b = {k: v for k, v in a.items() if k not in ("new_lengths", "num_tokens")}
    with pytest.raises(TypeError, match="bool"):
        release_pages(finished=torch.zeros(3, dtype=i32), **b)
    with pytest.raises(RuntimeError, match="sm_100"):
        release_pages(finished=torch.zeros(3, dtype=torch.bool), **b)


def test_cache_constructor():
    with pytest.raises(ValueError, match="page_size"):
        PagedKVCache(4, 0, 2, 64, 3, 2, device="cpu", dtype=torch.float16)
    with pytest.raises(ValueError, match="layers"):
        PagedKVCache(4, 16, 2, 64, 3, 2, layers=True, device="cpu", dtype=torch.float16)
    c = kotflash.PagedKVCache(4, 16, 2, 64, 3, 2, layers=5, device="cpu", dtype=torch.float16)
    assert c.k.shape == (5, 4, 2, 16, 64) and c.free_pages.tolist() == [3, 2, 1, 0] and c.free_count.tolist() == [4]
    assert c.block_table.tolist() == [[-1, -1]] * 3 and c.lengths.tolist() == [0] * 3


def _t(shape, ptr=0x1000, strides=None):
    if shape is None:
        return (0,) * 9
    return (ptr, *shape, *(strides or [shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1]))


def test_structs_have_the_headers_sizes(tmp_path):
    """The packed layouts against sizeof of the C structs and the offset of their last fields."""
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    root = Path(__file__).resolve().parents[1]
    names = [("decode", "stream"), ("append", "stream"), ("reserve", "starts"), ("release", "finished")]
    (tmp_path / "s.c").write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"kotflash_b200.h\"\nint main(void) {"
                                  + "".join(f'printf("%zu %zu\\n", sizeof(kf_paged_{n}_args), offsetof(kf_paged_{n}_args, {last}));'
                                            for n, last in names) + "return 0; }")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(root / "include"), str(tmp_path / "s.c"), "-o",
                    str(tmp_path / "s")], check=True, capture_output=True, text=True)
    lines = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()
    assert _ext.pack_paged_step.__self__.size == _ext.pack_paged_decode.__self__.size
    for i, (n, _) in enumerate(names):
        size = getattr(_ext, f"pack_paged_{n}").__self__.size
        assert int(lines[2 * i]) == size and int(lines[2 * i + 1]) == size - 8


def test_c_abi_refuses_before_any_launch():
    lib = _ext.load()
    p = 0x1000

    def decode(q=(3, 4, 1, 64), k=(5, 2, 16, 64), v=None, o=p, table=p, max_pages=2, lens=p, nk=None, nv=None, slots=0,
               dtype=0, ws=0, ws_bytes=0, q_strides=None, k_ptr=p):
        rows = (*_t(nk), *_t(nv), slots)
        pack, rows = (_ext.pack_paged_step, rows) if any(rows) else (_ext.pack_paged_decode, ())
        return lib.kf_paged_decode(pack(*_t(q, strides=q_strides), *_t(k, k_ptr), *_t(v or k), *rows, table, max_pages,
                                        max_pages, lens, o, 0, dtype, 0.1, ws, ws_bytes, 0, 0))

    for kw, code, match in [
        (dict(dtype=5), _ext.KF_ERR_INVALID, "dtype"),
        (dict(v=(5, 2, 16, 72)), _ext.KF_ERR_INVALID, "K/V page shapes"),
        (dict(o=0), _ext.KF_ERR_INVALID, "null data"),
        (dict(o=0x1008), _ext.KF_ERR_INVALID, "16-byte"),
        (dict(q=(3, 4, 2, 64)), _ext.KF_ERR_INVALID, "one token"),
        (dict(q=(3, 5, 1, 64)), _ext.KF_ERR_INVALID, "divisible"),
        (dict(q=(3, 4, 1, 72)), _ext.KF_ERR_INVALID, "head dimensions"),
        (dict(q=(3, 4, 1, 20), k=(5, 2, 16, 20)), _ext.KF_ERR_UNSUPPORTED, "multiple of 8"),
        (dict(q=(3, 4, 1, 136), k=(5, 2, 16, 136)), _ext.KF_ERR_UNSUPPORTED, "multiple of 8"),
        (dict(k=(0, 2, 16, 64)), _ext.KF_ERR_INVALID, "non-zero"),
        (dict(max_pages=0), _ext.KF_ERR_INVALID, "non-zero"),
        (dict(k=(5, 2, 1 << 21, 64)), _ext.KF_ERR_UNSUPPORTED, "too large"),
        (dict(q_strides=[256, 68, 68, 1]), _ext.KF_ERR_INVALID, "16-byte"),
        (dict(k_ptr=0x1008), _ext.KF_ERR_INVALID, "16-byte"),
        (dict(table=0), _ext.KF_ERR_INVALID, "null data"),
        (dict(nk=(3, 2, 1, 64)), _ext.KF_ERR_INVALID, "go together"),
        (dict(nk=(3, 2, 1, 64), nv=(3, 2, 1, 64)), _ext.KF_ERR_INVALID, "go together"),
        (dict(nk=(3, 2, 2, 64), nv=(3, 2, 2, 64), slots=p), _ext.KF_ERR_INVALID, "new K/V must be"),
        (dict(nk=(3, 2, 1, 64), nv=(3, 2, 1, 72), slots=p), _ext.KF_ERR_INVALID, "new K and V shapes"),
        (dict(max_pages=100), _ext.KF_ERR_WORKSPACE, "workspace needs"),
    ]:
        assert decode(**kw) == code, kw
        assert match in _ext.last_error(), (kw, _ext.last_error())
    assert lib.kf_paged_decode(None) == _ext.KF_ERR_INVALID

    def append(k=(5, 2, 16, 64), nk=(1, 2, 3, 64), nv=None, slots=p, dtype=1):
        return lib.kf_paged_append(_ext.pack_paged_append(*_t(k), *_t(k), *_t(nk), *_t(nv or nk), slots, dtype, 0))

    for kw, match in [(dict(nk=(1, 3, 3, 64)), "heads"), (dict(nv=(1, 2, 4, 64)), "new K/V shapes"), (dict(slots=0), "null"),
                      (dict(dtype=9), "dtype"), (dict(nk=(1, 2, 0, 64)), "non-zero")]:
        assert append(**kw) == _ext.KF_ERR_INVALID, kw
        assert match in _ext.last_error()

    def tables(B=3, max_pages=4, stride=4, pages=9, page=16, lens=p, out=p):
        return (lens, B, p, max_pages, stride, p, pages, p, page, out, p, 0)

    def reserve(slots=p, n=8, per=0, starts=p, **kw):
        return lib.kf_paged_reserve(_ext.pack_paged_reserve(*tables(**kw), p, slots, n, per, starts))

    def release(finished=p, **kw):
        return lib.kf_paged_release(_ext.pack_paged_release(*tables(**kw), finished))

    for call, kw, code, match in [
        (reserve, dict(B=0), _ext.KF_ERR_INVALID, "non-zero"), (reserve, dict(page=0), _ext.KF_ERR_INVALID, "page_size"),
        (reserve, dict(stride=3), _ext.KF_ERR_INVALID, "overlap"), (reserve, dict(B=20000), _ext.KF_ERR_UNSUPPORTED, "requests"),
        (reserve, dict(n=-1), _ext.KF_ERR_INVALID, "num_tokens"), (reserve, dict(per=2), _ext.KF_ERR_INVALID, "tokens_per_request"),
        (reserve, dict(slots=0), _ext.KF_ERR_INVALID, "null"), (reserve, dict(slots=0x1008), _ext.KF_ERR_INVALID, "16-byte"),
        (reserve, dict(starts=0), _ext.KF_ERR_INVALID, "null"), (reserve, dict(lens=0), _ext.KF_ERR_INVALID, "null"),
        (release, dict(pages=0), _ext.KF_ERR_INVALID, "non-zero"), (release, dict(out=0), _ext.KF_ERR_INVALID, "null"),
        (release, dict(finished=0), _ext.KF_ERR_INVALID, "null"),
        (release, dict(pages=2**31), _ext.KF_ERR_UNSUPPORTED, "too many pages"),
    ]:
        assert call(**kw) == code, kw
        assert match in _ext.last_error(), (kw, _ext.last_error())


def test_workspace_grows_with_the_row_tiles():
    lib = _ext.load()
    sizes = [lib.kf_paged_decode_workspace_bytes(g * 4, 4, 128, 148) for g in (1, 8, 9, 16, 17, 32, 33, 64, 65, 300)]
    assert sizes == sorted(sizes) and sizes[0] >= 148 * 2 * 2 * 8 * 129 * 4
    assert lib.kf_paged_decode_workspace_bytes(0, 4, 128, 148) == 0


def _walk(lens, units, tile, grid):
    """The kernel's walk over its list, in which a unit has a position for each
    tile and one for its end: every unit is finished once, whole or from
    partials that cover its tiles in order and use each slot once."""
    tiles = [(max(0, n) + tile - 1) // tile for n in lens]
    flat = [(b, h, x) for b in range(len(lens)) if tiles[b] for h in range(units) for x in range(tiles[b] + 1)]
    shares = min(grid, len(flat))
    done, parts, joins, tiles_done = set(), {}, {}, set()
    even, longer = (len(flat) // shares, len(flat) % shares) if shares else (0, 0)
    covered = 0
    for me in range(shares):
        begin = me * even + min(me, longer)
        end = begin + even + (1 if me < longer else 0)
        assert end > begin == covered
        covered = end
        pos = begin
        if flat[pos][2] == tiles[flat[pos][0]]:  # a unit's end comes first
            if begin + 1 >= end:
                continue
            pos += 1
        unit_t0 = flat[pos][2]
        going = True
        while going:
            b, h, x = flat[pos]
            assert x < tiles[b] and pos < end and (b, h, x) not in tiles_done
            tiles_done.add((b, h, x))
            unit_done = x + 1 == tiles[b]
            following = pos + (2 if unit_done else 1)
            going = following < end
            if unit_done or not going:
                if unit_t0 == 0 and unit_done:
                    assert (b, h) not in done
                    done.add((b, h))
                else:
                    slot = (me, 0 if unit_t0 > 0 else 1)
                    assert slot not in parts
                    parts[slot] = (b, h, unit_t0, x)
                    if unit_t0 == 0:
                        last = pos + (tiles[b] - 1 - x)
                        in_longer = longer * (even + 1)
                        joins[me] = (b, h, last // (even + 1) if last < in_longer else longer + (last - in_longer) // even)
                unit_t0 = 0
            pos = following
    assert covered == len(flat) and len(tiles_done) == units * sum(tiles)
    for me, (b, h, last_share) in joins.items():
        assert (b, h) not in done
        done.add((b, h))
        at = 0
        for j in range(last_share - me + 1):
            pb, ph, first, last = parts.pop((me + j, 1 if j == 0 else 0))
            assert (pb, ph, first) == (b, h, at)
            at = last + 1
        assert at == tiles[b]
    assert not parts and len(done) == units * sum(1 for t in tiles if t)


def test_work_split_covers_every_unit_once():
    r = random.Random(0)
    for _ in range(600):
        lens = [r.choice([0, 1, r.randint(0, 100), r.randint(0, 3000)]) for _ in range(r.randint(1, 12))]
        _walk(lens, r.randint(1, 6), r.choice([32, 64, 128]), r.randint(1, 60))


def test_oracle_attention_by_differences_of_order():
    """The oracle on a case small enough to write out: two positions, one masked page."""
    q = torch.tensor([[[[1.0, 0.0]]]])
    k = torch.tensor([[[[1.0, 5.0], [9.0, 9.0]]], [[[2.0, -5.0], [9.0, 9.0]]]])
    v = torch.tensor([[[[1.0, 10.0], [9.0, 9.0]]], [[[3.0, 20.0], [9.0, 9.0]]]])
    table = torch.tensor([[0, -1, 1]], dtype=torch.int32)
    o, lse, _ = oracle.attention(q, k, v, table, torch.tensor([5], dtype=torch.int32), 1.0)
    x = torch.tensor([1.0, 9.0, 2.0], dtype=torch.float64)  # page 0 rows 0, 1, then page 1 row 0
    w = torch.softmax(x, 0)
    assert torch.allclose(o[0, 0, 0], w[0] * v[0, 0, 0].double() + w[1] * v[0, 0, 1].double() + w[2] * v[1, 0, 0].double())
    assert torch.allclose(lse[0, 0], torch.logsumexp(x, 0))
