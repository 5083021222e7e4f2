"""Sizes that no launch holds are refused before anything runs.  No GPU needed."""
import ctypes

import pytest

from ratchet_amd import _lib

SOME, NO_DEVICE, SIZE = ctypes.c_void_p(0x1000), 8, 6


@pytest.mark.parametrize("seqs, kv_heads, head_dim, status", [(65535, 127, 8, NO_DEVICE), (65535, 129, 8, SIZE), (65535, 64, 2048, NO_DEVICE), (65535, 33, 8192, SIZE)])
def test_evict_of_more_rows_than_a_launch_holds(seqs, kv_heads, head_dim, status):
    """two blocks at least to a sequence, KV head and 4 KiB of a row, of which a launch holds 2^24 - 1"""
    kv = _lib.PagedKV(0x1000, 0x2000, 0x3000, 0x4000, 10, kv_heads, 4, head_dim, seqs, 3)
    lib = _lib.load()
    for table_out in (SOME, ctypes.c_void_p(0x3000)):
        assert lib.rt_paged_evict(None, 2, kv, SOME, 5, 1, 1, table_out, SOME, SOME) == status, lib.rt_last_error()
