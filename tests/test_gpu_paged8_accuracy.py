# SPDX-License-Identifier: Apache-2.0
"""How far what the 8-bit paged cache gives back is from what it was given:
the bounds of ``kotflash_b200.paged8``, also after a scale has grown (GPU)."""
import pytest
import torch

from kotflash_b200 import append_paged_kv8, read_paged_kv8

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _pool(n, hkv, page, d, block, held):
    codes = [torch.zeros(n, hkv, page, d, dtype=torch.uint8, device="cuda").view(FORMATS[held]) for _ in range(2)]
    scales = [torch.zeros(n, hkv, page // block, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    return (*codes, *scales)


def _scales(scales, page):
    raw = scales.view(torch.uint8).double()
    return torch.exp2(raw - 127).repeat_interleave(page // scales.shape[2], 2)  # [pages, Hkv, page]


def _bound(x, scale, held, grown):
    """Rounded once: half a step, 2^-4 of an e4m3 element or, of a subnormal
    one, 2^-10 of the scale; half of an int8 scale.  Rounded again as the scale
    grew, at least by two each time: e4m3 codes that stay normal are exact, others are off by 2^-10
    of each scale more, in all less than 2^-9 of the last; int8 by half of each,
    in all less than the last."""
    if held == "int8":
        return scale * (1.0 if grown else 0.5)
    once = torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    return x.abs() * 2.0 ** -4 + scale * 2.0 ** -9 if grown else once


@pytest.mark.parametrize("held", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("block", [1, 2, 16])
def test_rows_whose_scale_grows_later(held, dtype, block):
    """Tokens one by one, each up to 2.2 times the ones before: a scale grows
    up to 15 times under its first rows."""
    page, hkv, d, n = 16, 2, 64, 4
    cache = _pool(n, hkv, page, d, block, held)
    g = torch.Generator(device="cuda").manual_seed(block)
    size = torch.exp2(torch.arange(page, device="cuda") * 1.1 - 10)[:, None, None] * (0.2 + torch.rand(page, n, hkv, device="cuda", generator=g))
    rows = (torch.randn(2, page, n, hkv, d, device="cuda", generator=g) * size[..., None]).to(dtype)
    rows[:, :, :, :, 5] = 1.4995
    for i in range(page):
        new = rows[:, i, None].transpose(2, 3).contiguous()  # [2, 1, Hkv, n, D]
        append_paged_kv8(*cache, new[0], new[1], torch.arange(n, device="cuda") * page + i)
    back = read_paged_kv8(*cache, torch.arange(n * page, device="cuda"), dtype=BF16)
    for got, given, scales in zip(back, rows, cache[2:]):
        got = got[0].view(hkv, n, page, d).permute(2, 1, 0, 3).double()
        scale = _scales(scales, page).permute(2, 0, 1)[..., None]
        assert ((got - given.double()).abs() <= _bound(given.double(), scale, held, block > 1)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_the_largest_step_of_int8(dtype):
    """A largest element that just does not round to 127 takes twice the scale,
    2 / 127.5 of it: an element of half of that is lost, and none is off by more."""
    cache = _pool(1, 1, 16, 64, 1, "int8")
    x = torch.zeros(1, 1, 3, 64, device="cuda", dtype=dtype)
    x[..., 0] = torch.tensor([127.0, 127.5, 128.0], device="cuda")
    x[..., 1:] = torch.linspace(-1.5, 1.5, 63, device="cuda").to(dtype)
    append_paged_kv8(*cache, x, x, torch.arange(3, device="cuda"))
    k, _ = read_paged_kv8(*cache, torch.arange(3, device="cuda"), dtype=dtype)
    off = (k.double() - x.double()).abs()
    top = x.double().abs().amax(-1, keepdim=True)
    assert (off <= top / 127.5).all()
    # 127 is held under a scale of 1; 127.5, a tie, rounds to 128 (in bf16 the number is 128 to begin with)
    assert cache[2].view(torch.uint8).flatten()[:3].tolist() == [127, 128, 128]
    assert off[0, 0, 0].max() <= 0.5 and off[0, 0, 1:].max() > 0.9


@pytest.mark.parametrize("held", ["e4m3", "int8"])
def test_rows_below_the_smallest_scale(held):
    """Where 2^-60 is the scale, an element is off by half of an int8 step of it, 2^-10 of it in e4m3 or 2^-4 of itself."""
    cache = _pool(1, 1, 16, 64, 1, held)
    x = (torch.randn(1, 1, 8, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
         * torch.exp2(-torch.arange(8, device="cuda").float() * 2 - 52)[:, None]).to(BF16)
    append_paged_kv8(*cache, x, x, torch.arange(8, device="cuda"))
    k, _ = read_paged_kv8(*cache, torch.arange(8, device="cuda"), dtype=BF16)
    scale = _scales(cache[2], 16).view(1, 1, 16)[..., :8, None]
    assert ((k.double() - x.double()).abs() <= _bound(x.double(), scale, held, False)).all()
