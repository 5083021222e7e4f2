"""Arguments that the Python layer of attention and the cache refuses before the library sees them.  No GPU needed."""
import ctypes
import math

import pytest

from ratchet_amd import _lib
from ratchet_amd.runtime import Device, PagedCache


class Shape:
    """stands for a buffer: its shape and type are what is looked at"""

    def __init__(self, shape, dt):
        self.shape, self.dt, self.ptr, self.numel = shape, dt, ctypes.c_void_p(0x1000), math.prod(shape)


class Library:
    """stands for the library: counts the calls that reach it"""

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def call(*args):
            self.calls += 1
            return 0
        return call


@pytest.fixture
def dev():
    d = Device.__new__(Device)
    d.lib, d.handle = Library(), None
    yield d
    d.handle = None


Q, K = Shape((1, 4, 8, 64), _lib.F16), Shape((1, 2, 20, 64), _lib.F16)
CACHE = PagedCache(Shape((9, 2, 16, 64), _lib.F16), Shape((9, 2, 16, 64), _lib.F16), Shape((3, 5), _lib.I32), Shape((3,), _lib.I32))
ROWS, TOKENS, STARTS, WEIGHTS = Shape((6, 2, 64), _lib.F16), Shape((6, 4, 64), _lib.F16), Shape((4,), _lib.I32), Shape((3, 2, 80), _lib.F32)


def attention(dev, **change):
    return dev.attention(**{**dict(q=Q, k=K, v=K, out=Q), **change})


def append(dev, **change):
    return dev.paged_append(CACHE, **{**dict(starts=STARTS, k=ROWS, v=ROWS), **change})


def paged(dev, **change):
    return dev.paged_attention(cache=CACHE, **{**dict(q=TOKENS, starts=STARTS, out=TOKENS), **change})


def test_calls_that_reach_the_library(dev):
    attention(dev, q_strides=(2048, 512, 64, 1), k_strides=(2560, 1280, 64, 1), v_strides=[0, 0, 0, 1], out_strides=(2048, 512, 64, 1))
    append(dev, k_strides=(128, 64), v_strides=[0, 64])
    paged(dev, q_strides=(256, 64))
    assert dev.lib.calls == 3


@pytest.mark.parametrize("call, name, strides", [
    *[(attention, name, s) for name in ("q_strides", "k_strides", "v_strides", "out_strides") for s in ((), (64,), (512, 64, 1), (0, 0, 0, 0, 1))],
    *[(append, name, s) for name in ("k_strides", "v_strides") for s in ((), (128,), (128, 64, 1), (128, 64, 2))],
    *[(paged, "q_strides", s) for s in ((), (256,), (256, 64, 1), (64, 64, 2))],
])
def test_another_number_of_strides_than_the_library_reads(dev, call, name, strides):
    with pytest.raises(ValueError, match="strides"):
        call(dev, **{name: strides})
    assert dev.lib.calls == 0


def evict(dev, **change):
    return dev.paged_evict(CACHE, **{**dict(weights=WEIGHTS, keep=40), **change})


@pytest.mark.parametrize("call, name, value", [
    *[(call, name, v) for call in (attention, paged) for name in ("window", "sinks") for v in (-1, -5, 2 ** 32, 2 ** 32 + 7)],
    *[(evict, name, v) for name in ("keep", "first", "recent") for v in (-1, -(2 ** 32) + 3, 2 ** 32, 2 ** 32 + 7)],
])
def test_counts_that_32_bits_do_not_hold(dev, call, name, value):
    """taken modulo 2^32 they would be other counts: -1 sinks all keys, 2^32 + 7 a window of 7"""
    with pytest.raises(ValueError, match=name):
        call(dev, **{name: value})
    assert dev.lib.calls == 0


def test_counts_that_32_bits_hold(dev):
    attention(dev, window=2 ** 32 - 1, sinks=2 ** 32 - 1)
    paged(dev, window=2 ** 32 - 1, sinks=0)
    evict(dev, keep=80, first=0, recent=80)
    assert dev.lib.calls == 3
