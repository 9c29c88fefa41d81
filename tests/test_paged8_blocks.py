# SPDX-License-Identifier: Apache-2.0
"""The 8-bit paged cache with several tokens to a scale, on the CPU."""
from kotflash_b200 import _ext


def test_pools_of_more_blocks_than_memory_holds_are_refused():
    """Stores tell blocks apart by 32 bits."""
    p, pages, page = 0x1000, 2 ** 31 - 1, 64
    pool = (p, pages, 1, page, 16, page * 16, page * 16, 16, 1)
    rows = (p, 1, 1, 3, 16, 48, 48, 16, 1)
    args = _ext.pack_paged8_append(*pool, *pool, p, p, 32, 32, 32, 32, 2, 0, *rows, *rows, p, 0, 0)
    assert _ext.load().kf_paged8_append(args) == _ext.KF_ERR_UNSUPPORTED and "too large" in _ext.last_error()
