# SPDX-License-Identifier: Apache-2.0
"""The 8-bit paged KV cache on the CPU: its format, the refusals of the Python
layer and of the C ABI (before any launch)."""
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import kotflash_b200 as kotflash
from kotflash_b200 import _ext, append_paged_kv8, paged_attention8, read_paged_kv8
from oracle import paged8_oracle as oracle

F16, F8, E8 = torch.float16, torch.float8_e4m3fn, torch.float8_e8m0fnu


# ---------------------------------------------------------------- the format

def test_oracle_rounds_as_the_types_do():
    x = torch.randn(20000, dtype=torch.float64, generator=torch.Generator().manual_seed(1)) * torch.logspace(-4, 2, 20000, dtype=torch.float64)
    x = torch.cat((x.clamp(-448, 448), torch.arange(-448, 449).double() / 2, torch.arange(0, 64).double() / 1024))
    assert torch.equal(oracle.round_code(x, "e4m3"), x.float().to(F8).double())
    assert torch.equal(oracle.round_code(x, "int8"), torch.round(x))


@pytest.mark.parametrize("held,largest", [("e4m3", 448.0), ("int8", 127.0)])
def test_oracle_scales_are_the_smallest_that_hold(held, largest):
    for top in (1e-30, 2.0 ** -70, 1e-3, 0.5, 1.0, 127.0, 127.4, 127.5, 128.0, 448.0, 449.0, 3e4, 65504.0, 1e18):
        e = oracle.exponent(top, held)
        code = abs(oracle.round_code(torch.tensor([top / 2.0 ** e], dtype=torch.float64), held).item())
        assert code <= largest
        if e > -60:
            below = top / 2.0 ** (e - 1)
            assert (below > 448) if held == "e4m3" else (round(below) > 127)
    assert oracle.exponent(0.0, held) == -60
    assert all(math.isnan(oracle.exponent(x, held)) for x in (math.inf, math.nan, 1e30))


def test_oracle_keeps_what_a_growing_scale_allows():
    codes, exps = torch.zeros(1, 1, 4, 2, dtype=torch.float64), torch.zeros(1, 1, 1, dtype=torch.float64)
    oracle.store(codes, exps, torch.tensor([[[[100.0, 3.0]]]]), [0], "int8")
    oracle.store(codes, exps, torch.tensor([[[[254.0, 1.0]]]]), [1], "int8")
    assert exps.item() == 1 and codes[0, 0, :2].tolist() == [[50, 2], [127, 0]]
    oracle.store(codes, exps, torch.tensor([[[[1.0, 1.0]]]]), [2], "int8")
    assert exps.item() == 1 and codes[0, 0, 2].tolist() == [0, 0]
    oracle.store(codes, exps, torch.tensor([[[[1.0, 1.0]]]]), [0], "int8")      # begun anew
    assert exps.item() == -6 and codes[0, 0, 0].tolist() == [64, 64]


# ---------------------------------------------------------------- refusals

def _cache(held=F8, d=64, page=16, block=1, pages=5, hkv=2):
    p = torch.zeros(pages, hkv, page, -(-d // 16) * 16, dtype=torch.uint8).view(held)[..., :d]
    s = torch.zeros(pages, hkv, page // block, dtype=torch.uint8).view(E8)
    return dict(k_pages=p, v_pages=p.clone() if d % 16 == 0 else p, k_scales=s, v_scales=s.clone())


def _attend_args(**changes):
    a = dict(q=torch.zeros(3, 4, 1, 64, dtype=F16), **_cache(), block_table=torch.zeros(3, 2, dtype=torch.int32),
             lengths=torch.zeros(3, dtype=torch.int32))
    a.update(changes)
    return a


_ROW = torch.zeros(3, 2, 1, 64, dtype=F16)


@pytest.mark.parametrize("changes,error,match", [
    (dict(q=None), TypeError, "torch.Tensor"),
    (dict(k_pages=None), TypeError, "torch.Tensor"),
    (dict(k_pages=torch.zeros(5, 2, 16, 64, dtype=F16)), TypeError, "float8_e4m3fn or int8"),
    (dict(v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.int8)), ValueError, "one dtype"),
    (dict(k_scales=torch.zeros(5, 2, 16, dtype=torch.uint8)), TypeError, "float8_e8m0fnu"),
    (dict(k_scales=torch.zeros(5, 2, 8, dtype=torch.uint8).view(E8)), ValueError, "scales must be"),
    (_cache(page=16, block=16) | dict(k_scales=torch.zeros(5, 2, 3, dtype=torch.uint8).view(E8), v_scales=torch.zeros(5, 2, 3, dtype=torch.uint8).view(E8)),
     ValueError, "scales must be"),
    (dict(v_pages=torch.zeros(5, 2, 8, 64, dtype=torch.uint8).view(F8)), ValueError, "shapes must match"),
    (dict(k_scales=torch.zeros(5, 2, 32, dtype=torch.uint8).view(E8)[..., ::2], v_scales=torch.zeros(5, 2, 16, dtype=torch.uint8).view(E8)),
     ValueError, "contiguous"),
    (dict(q=torch.zeros(3, 4, 1, 64)), TypeError, "float16 and bfloat16"),
    (dict(q=torch.zeros(3, 4, 64, dtype=F16)), ValueError, "4-D"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), TypeError, "lengths must be int32"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "block_table must be"),
    (dict(lengths=torch.zeros(6, dtype=torch.int32)[::2]), ValueError, "lengths must be"),
    (dict(q=torch.zeros(3, 5, 1, 64, dtype=F16)), ValueError, "divisible"),
    (dict(q=torch.zeros(3, 0, 1, 64, dtype=F16)), ValueError, "non-zero"),
    (dict(new_k=_ROW), ValueError, "go together"),
    (dict(slots=torch.zeros(3, dtype=torch.int64)), ValueError, "go together"),
    (dict(new_k=_ROW, new_v=_ROW.bfloat16(), slots=torch.zeros(3, dtype=torch.int64)), ValueError, "dtypes must match"),
    (dict(new_k=_ROW, new_v=_ROW, slots=torch.zeros(3, dtype=torch.int32)), TypeError, "slots must be int64"),
    (dict(scale="x"), TypeError, "scale"),
    (dict(scale=float("nan")), ValueError, "finite"),
    (dict(q=torch.zeros(3, 4, 1, 64, dtype=F16, requires_grad=True)), RuntimeError, "inference-only"),
    (dict(), RuntimeError, "sm_100"),
])
def test_attention_refusals(changes, error, match):
    with pytest.raises(error, match=match):
        paged_attention8(**_attend_args(**changes))


def test_append_and_read_refusals():
    rows, slots = torch.zeros(1, 2, 3, 64, dtype=F16), torch.zeros(3, dtype=torch.int64)
    cache = _cache()
    for more, error, match in [
        (dict(slots=slots.int()), TypeError, "int64"), (dict(slots=slots[:2]), ValueError, "one slot for each"),
        (dict(new_v=rows.bfloat16()), ValueError, "dtypes"), (dict(new_k=rows.float()), TypeError, "float16 and bfloat16"),
        (dict(new_k=rows[0]), ValueError, "4-D"), (dict(new_k=None), TypeError, "torch.Tensor"),
        (dict(new_k=rows.clone().requires_grad_(True)), RuntimeError, "inference-only"), (dict(), RuntimeError, "sm_100"),
    ]:
        with pytest.raises(error, match=match):
            append_paged_kv8(**(cache | dict(new_k=rows, new_v=rows, slots=slots) | more))
    for more, error, match in [
        (dict(slots=slots.int()), TypeError, "int64"), (dict(slots=slots[None]), ValueError, "slots must be"),
        (dict(dtype=torch.float32), TypeError, "float16 and bfloat16"), (dict(slots=None), TypeError, "torch.Tensor"),
        (dict(), RuntimeError, "sm_100"),
    ]:
        with pytest.raises(error, match=match):
            read_paged_kv8(**(cache | dict(slots=slots, dtype=F16) | more))


def test_cache_constructor():
    for kw, error, match in [
        (dict(dtype=F16), TypeError, "float8_e4m3fn or int8"), (dict(scale_block=3), ValueError, "scale_block"),
        (dict(scale_block=32), ValueError, "scale_block"), (dict(scale_block=True), ValueError, "scale_block"),
        (dict(layers=0), ValueError, "layers"),
    ]:
        with pytest.raises(error, match=match):
            kotflash.PagedKVCache8(4, 16, 2, 64, 3, 2, device="cpu", **kw)
    c = kotflash.PagedKVCache8(4, 16, 2, 72, 3, 2, layers=5, scale_block=8, device="cpu", dtype=torch.int8)
    assert c.k.shape == (5, 4, 2, 16, 72) and c.k.stride(3) == 80 and c.k.dtype == torch.int8
    assert c.v_scales.shape == (5, 4, 2, 2) and c.v_scales.dtype == E8
    assert c.free_pages.tolist() == [3, 2, 1, 0] and c.block_table.tolist() == [[-1, -1]] * 3
    assert kotflash.PagedKVCache8(4, 16, 2, 64, 3, 2, device="cpu").k.dtype == F8


# ---------------------------------------------------------------- the C ABI

def test_structs_have_the_headers_sizes(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    root = Path(__file__).resolve().parents[1]
    names = [("paged8_append", "stream"), ("paged8_read", "stream"), ("paged8_decode", "stream"), ("rotary", "stream")]
    (tmp_path / "s.c").write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"kotflash_b200.h\"\nint main(void) {"
                                  + "".join(f'printf("%zu %zu\\n", sizeof(kf_{n}_args), offsetof(kf_{n}_args, {last}));'
                                            for n, last in names)
                                  + 'printf("%zu\\n", offsetof(kf_paged8_decode_args, slots)); return 0; }')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(root / "include"), str(tmp_path / "s.c"), "-o",
                    str(tmp_path / "s")], check=True, capture_output=True, text=True)
    out = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()
    packs = [_ext.pack_paged8_append, _ext.pack_paged8_append, _ext.pack_paged8_decode, _ext.pack_rotary]
    for i, pack in enumerate(packs):
        assert int(out[2 * i]) == pack.__self__.size and int(out[2 * i + 1]) == pack.__self__.size - 8
    assert _ext.pack_paged8_step.__self__.size == _ext.pack_paged8_decode.__self__.size


P = 0x1000


def _t(shape, ptr=P, strides=None):
    if shape is None:
        return (0,) * 9
    return (ptr, *shape, *(strides or [shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1]))


def _c(k=(5, 2, 16, 64), v=None, ks=P, vs=P, block=1, form=0, ptr=P, strides=None):
    return (*_t(k, ptr, strides), *_t(v or k, P, strides), ks, vs, 32, 16, 32, 16, block, form)


CACHE_FAULTS = [
    (dict(form=2), _ext.KF_ERR_INVALID, "e4m3 or int8"), (dict(v=(5, 2, 8, 64)), _ext.KF_ERR_INVALID, "K/V page shapes"),
    (dict(k=(0, 2, 16, 64)), _ext.KF_ERR_INVALID, "non-zero"), (dict(ks=0), _ext.KF_ERR_INVALID, "null"),
    (dict(block=3), _ext.KF_ERR_INVALID, "power of two"), (dict(block=32), _ext.KF_ERR_INVALID, "power of two"),
    (dict(block=0), _ext.KF_ERR_INVALID, "power of two"), (dict(ptr=0x1008), _ext.KF_ERR_INVALID, "16-byte"),
    (dict(strides=[2048, 1024, 72, 1]), _ext.KF_ERR_INVALID, "16-byte"), (dict(strides=[2048, 1024, 64, 2]), _ext.KF_ERR_INVALID, "16-byte"),
    (dict(strides=[2048, 1024, -64, 1]), _ext.KF_ERR_INVALID, "16-byte"), (dict(k=(5, 2, 1 << 21, 64)), _ext.KF_ERR_UNSUPPORTED, "too large"),
]


def _refused(rc, code, match, kw):
    assert rc == code, (kw, rc, _ext.last_error())
    assert match in _ext.last_error(), (kw, _ext.last_error())


def test_c_abi_store_and_load_refuse_before_any_launch():
    lib = _ext.load()

    def move(fn, rows=(1, 2, 3, 64), row_v=None, slots=P, dtype=1, row_ptr=P, row_strides=None, **kw):
        return fn(_ext.pack_paged8_append(*_c(**kw), *_t(rows, row_ptr, row_strides), *_t(row_v or rows, P, row_strides), slots, dtype, 0))

    for fn in (lib.kf_paged8_append, lib.kf_paged8_read):
        for kw, code, match in CACHE_FAULTS + [
            (dict(dtype=7), _ext.KF_ERR_INVALID, "dtype"), (dict(rows=(1, 3, 3, 64)), _ext.KF_ERR_INVALID, "heads and head_dim"),
            (dict(rows=(1, 2, 3, 72)), _ext.KF_ERR_INVALID, "heads and head_dim"), (dict(row_v=(1, 2, 4, 64)), _ext.KF_ERR_INVALID, "must match"),
            (dict(rows=(1, 2, 0, 64)), _ext.KF_ERR_INVALID, "non-zero"), (dict(slots=0), _ext.KF_ERR_INVALID, "null"),
            (dict(row_ptr=0x1008), _ext.KF_ERR_INVALID, "16-byte"), (dict(row_strides=[384, 192, 68, 1]), _ext.KF_ERR_INVALID, "16-byte"),
            (dict(rows=(1, 2, 2 ** 28, 64)), _ext.KF_ERR_UNSUPPORTED, "too large"),
            (dict(k=(5, 2, 16, 20), rows=(1, 2, 3, 20)), _ext.KF_ERR_UNSUPPORTED, "multiple of 8"),
        ]:
            _refused(move(fn, **kw), code, match, kw)
        assert fn(None) == _ext.KF_ERR_INVALID


def test_c_abi_attention_refuses_before_any_launch():
    lib = _ext.load()

    def decode(q=(3, 4, 1, 64), o=P, table=P, max_pages=2, lens=P, nk=None, nv=None, slots=0, dtype=0, ws=0, ws_bytes=0,
               q_strides=None, scale=0.1, **kw):
        rows = (*_t(nk), *_t(nv), slots)
        pack, rows = (_ext.pack_paged8_step, rows) if any(rows) else (_ext.pack_paged8_decode, ())
        return lib.kf_paged8_decode(pack(*_c(**kw), *_t(q, strides=q_strides), *rows, table, max_pages, max_pages, lens, o, 0,
                                         dtype, scale, ws, ws_bytes, 0, 0))

    for kw, code, match in CACHE_FAULTS + [
        (dict(dtype=5), _ext.KF_ERR_INVALID, "dtype"), (dict(o=0), _ext.KF_ERR_INVALID, "null data"),
        (dict(o=0x1008), _ext.KF_ERR_INVALID, "16-byte"), (dict(q=(3, 4, 2, 64)), _ext.KF_ERR_INVALID, "one token"),
        (dict(q=(3, 5, 1, 64)), _ext.KF_ERR_INVALID, "divisible"), (dict(q=(3, 4, 1, 72)), _ext.KF_ERR_INVALID, "head dimensions"),
        (dict(q=(3, 4, 1, 136), k=(5, 2, 16, 136)), _ext.KF_ERR_UNSUPPORTED, "multiple of 8"), (dict(max_pages=0), _ext.KF_ERR_INVALID, "non-zero"),
        (dict(q_strides=[256, 68, 68, 1]), _ext.KF_ERR_INVALID, "16-byte"), (dict(table=0), _ext.KF_ERR_INVALID, "null data"),
        (dict(nk=(3, 2, 1, 64)), _ext.KF_ERR_INVALID, "go together"), (dict(nk=(3, 2, 1, 64), nv=(3, 2, 1, 64)), _ext.KF_ERR_INVALID, "go together"),
        (dict(nk=(3, 2, 2, 64), nv=(3, 2, 2, 64), slots=P), _ext.KF_ERR_INVALID, "new K/V must be"),
        (dict(nk=(3, 2, 1, 64), nv=(3, 2, 1, 72), slots=P), _ext.KF_ERR_INVALID, "new K and V shapes"),
        (dict(scale=1e39), _ext.KF_ERR_INVALID, "scale"), (dict(max_pages=100), _ext.KF_ERR_WORKSPACE, "workspace needs"),
    ]:
        _refused(decode(**kw), code, match, kw)
    assert lib.kf_paged8_decode(None) == _ext.KF_ERR_INVALID
