"""Caps as large as they may be, and just beyond.  No GPU needed."""
import ctypes

import pytest

from ratchet_amd import _lib

SOME, NO_DEVICE, ARG = ctypes.c_void_p(0x1000), 8, 7


@pytest.mark.parametrize("cap, status", [(1.17e38, NO_DEVICE), (1.19e38, ARG), (2.3e38, ARG), (2.4e38, ARG), (3.4e38, ARG)])
def test_caps_whose_double_is_no_f32(cap, status):
    """twice the cap, in units of ln 2, is a factor of the kernels' own"""
    u4 = lambda *v: (ctypes.c_uint32 * 4)(*v)        # noqa: E731
    scores, lib = _lib.Scores(cap, None, None, 0, None), _lib.load()
    assert lib.rt_attention_scored(None, _lib.F32, SOME, u4(1, 2, 5, 64), None, SOME, None, SOME, None, u4(1, 2, 5, 64), None, SOME, None, None, 1.0, 1, 0, 0, ctypes.byref(scores)) == status
    kv = _lib.PagedKV(0x1000, 0x2000, 0x3000, 0x4000, 10, 2, 16, 64, 3, 4)
    assert lib.rt_paged_attention_scored(None, _lib.F32, SOME, None, 5, 2, kv, SOME, SOME, None, 1.0, 0, 0, ctypes.byref(scores)) == status
