# SPDX-License-Identifier: Apache-2.0
"""Paged KV cache on the CPU: refusals at its edges, before any launch, and what its sources must not hold."""
import math
import re
from pathlib import Path

import pytest
import torch

from kotflash_b200 import _ext, append_paged_kv, paged, reserve_pages


def test_appending_no_tokens_is_checked_like_any_append():
    pool, slots = torch.zeros(5, 2, 16, 64, dtype=torch.float16), torch.zeros(0, dtype=torch.int64)
    rows = torch.zeros(1, 2, 0, 64, dtype=torch.float16)
    for args, error, match in [
        ((pool, pool, rows, rows, slots.int()), TypeError, "int64"),
        ((pool, pool, rows, rows, torch.zeros(1, dtype=torch.int64)), ValueError, "one slot for each"),
        ((pool, pool, rows, rows.bfloat16(), slots), ValueError, "dtypes"),
        ((pool, pool, rows, rows, slots), RuntimeError, "sm_100"),
    ]:
        with pytest.raises(error, match=match):
            append_paged_kv(*args)


def test_dependent_launches_read_no_memory_non_coherently():
    """A kernel launched as a programmatic dependent lives while its predecessor
    writes; the non-coherent load path is for memory that nobody writes while
    the kernel lives."""
    csrc = Path(__file__).resolve().parents[1] / "kotflash_b200" / "csrc"
    sources = [p for p in csrc.glob("*.cu") if "launch_dependent" in p.read_text()]
    assert {p.name for p in sources} >= {"decode.cu", "paged_cache.cu", "paged_decode.cu"}
    for path in sources:
        found = re.findall(r"__ldg\b|ld\.global\.nc|__restrict__", path.read_text())
        assert not found, (path.name, found)


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
def test_nothing_of_a_tracing_mode_stays(monkeypatch):
    """reserve_pages on tensors without memory (an export, a shape pass) leaves no
    tensor of that mode in the module for later calls."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode

    calls = []

    class Library:
        def __getattr__(self, name):
            return lambda args: calls.append(name) or 0

    monkeypatch.setattr(_ext, "load", Library)
    monkeypatch.setattr(paged, "_is_sm100", lambda index: True)
    monkeypatch.setattr(paged, "_raw_stream", lambda index: 0)
    for mode in (FakeTensorMode(), FakeTensorMode()):
        with mode:
            i32 = dict(dtype=torch.int32, device="cuda")
            lengths = torch.empty(3, **i32)
            slots, _, _, _ = reserve_pages(lengths, torch.empty(3, **i32), torch.empty(3, 4, **i32), torch.empty(9, **i32),
                                           torch.empty(1, **i32), page_size=16, num_tokens=6)
            assert isinstance(slots, FakeTensor) and slots.fake_mode is mode and slots.dtype is torch.int64
    assert calls == ["kf_paged_reserve"] * 2


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39, -3e38])
def test_c_abi_refuses_a_scale_that_single_precision_does_not_hold(scale):
    def t4(*shape):
        return (0x1000, *shape, shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1)

    args = _ext.pack_paged_decode(*t4(3, 4, 1, 64), *t4(5, 2, 16, 64), *t4(5, 2, 16, 64), 0x1000, 2, 2, 0x1000, 0x1000, 0, 0,
                                  scale, 0, 0, 0, 0)
    assert _ext.load().kf_paged_decode(args) == _ext.KF_ERR_INVALID and "scale" in _ext.last_error()
