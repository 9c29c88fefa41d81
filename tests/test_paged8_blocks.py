# SPDX-License-Identifier: Apache-2.0
"""The 8-bit paged cache with several tokens to a scale, on the CPU."""
import torch

from kotflash_b200 import _ext
from oracle import paged8_oracle as oracle


def test_pools_of_more_blocks_than_memory_holds_are_refused():
    """Stores tell blocks apart by 32 bits."""
    p, pages, page = 0x1000, 2 ** 31 - 1, 64
    pool = (p, pages, 1, page, 16, page * 16, page * 16, 16, 1)
    rows = (p, 1, 1, 3, 16, 48, 48, 16, 1)
    args = _ext.pack_paged8_append(*pool, *pool, p, p, 32, 32, 32, 32, 2, 0, *rows, *rows, p, 0, 0)
    assert _ext.load().kf_paged8_append(args) == _ext.KF_ERR_UNSUPPORTED and "too large" in _ext.last_error()


def test_an_element_that_is_rounded_twice():
    """1.4995 becomes 1 under a scale of 1 and, when that grows to 2, a tie that
    goes to 0: off by more than half of the scale that it ends under, by less
    than all of it."""
    codes, exps = torch.zeros(1, 1, 4, 2, dtype=torch.float64), torch.zeros(1, 1, 1, dtype=torch.float64)
    oracle.store(codes, exps, torch.tensor([[[[100.0, 1.4995]]]]), [0], "int8")
    assert exps.item() == 0 and codes[0, 0, 0].tolist() == [100, 1]
    oracle.store(codes, exps, torch.tensor([[[[128.0, 0.0]]]]), [1], "int8")
    assert exps.item() == 1 and codes[0, 0, 0].tolist() == [50, 0]
    off = abs(oracle.values(codes, exps)[0, 0, 0, 1].item() - 1.4995)
    assert 0.5 * 2 < off < 2
