"""What the attention and cache entry points refuse, before any HIP call; and what the Python layer refuses.  No GPU needed."""
import ctypes

import pytest

from ratchet_amd import _lib

SOME, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001)
OK_BUT_NO_DEVICE, NULL, DTYPE, SHAPE, SIZE, ARG, ALIGN = 8, 1, 2, 4, 6, 7, 9


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def u4(*v):
    return (ctypes.c_uint32 * 4)(*v)


def s(*v):
    return (ctypes.c_uint64 * len(v))(*v)


ATTENTION = dict(dt=_lib.F16, q=SOME, q_shape=u4(2, 8, 16, 64), q_strides=None, k=SOME, k_strides=None, v=SOME, v_strides=None, kv_shape=u4(2, 2, 100, 64), lens=None, y=SOME,
                 y_strides=None, lse=None, scale=0.125, causal=1, window=0, sinks=0)


@pytest.mark.parametrize("change, status", [
    ({}, OK_BUT_NO_DEVICE),
    ({"dt": _lib.I32}, DTYPE), ({"dt": 9}, DTYPE),
    ({"q_shape": None}, NULL), ({"kv_shape": None}, NULL), ({"q": None}, NULL), ({"k": None}, NULL), ({"v": None}, NULL), ({"y": None}, NULL),
    ({"q_shape": u4(2, 8, 0, 64)}, SHAPE), ({"kv_shape": u4(2, 2, 0, 64)}, SHAPE), ({"q_shape": u4(0, 8, 16, 64), "kv_shape": u4(0, 2, 100, 64)}, SHAPE),
    ({"kv_shape": u4(2, 3, 100, 64)}, SHAPE), ({"kv_shape": u4(1, 2, 100, 64)}, SHAPE), ({"kv_shape": u4(2, 2, 100, 32)}, SHAPE),
    ({"q_shape": u4(2, 8, 16, 513), "kv_shape": u4(2, 2, 100, 513)}, SIZE), ({"q_shape": u4(2, 8, 1 << 31, 64)}, SIZE), ({"kv_shape": u4(2, 2, 1 << 31, 64)}, SIZE),
    ({"q_shape": u4(70000, 8, 16, 64), "kv_shape": u4(70000, 2, 100, 64)}, SIZE),
    ({"causal": 2}, ARG), ({"causal": 0}, OK_BUT_NO_DEVICE), ({"causal": 0, "window": 5}, ARG), ({"causal": 0, "sinks": 5}, ARG),
    ({"scale": float("nan")}, ARG), ({"scale": float("inf")}, ARG), ({"scale": -1.0}, OK_BUT_NO_DEVICE),
    ({"q": ODD}, ALIGN), ({"k": ODD}, ALIGN), ({"v": ODD}, ALIGN), ({"y": ODD}, ALIGN), ({"lse": ctypes.c_void_p(0x1002)}, ALIGN), ({"lens": ctypes.c_void_p(0x1002)}, ALIGN),
    ({"q_strides": s(1, 1, 1, 2)}, ARG), ({"k_strides": s(0, 0, 0, 1)}, OK_BUT_NO_DEVICE), ({"v_strides": s(1, 1, 1, 0)}, ARG),
    ({"y_strides": s(8 * 16 * 64, 64, 8 * 64, 1)}, OK_BUT_NO_DEVICE), ({"y_strides": s(8 * 16 * 64, 64, 8 * 64 - 1, 1)}, ARG), ({"y_strides": s(0, 16 * 64, 64, 1)}, ARG),
    ({"y_strides": s(8 * 16 * 64, 16 * 64, 63, 1)}, ARG), ({"k_strides": s(1 << 41, 64, 64, 1)}, SIZE), ({"k_strides": s((1 << 64) - 1, 64, 64, 1)}, SIZE),
    ({"window": (1 << 32) - 1, "sinks": (1 << 32) - 1}, OK_BUT_NO_DEVICE),
])
def test_attention(lib, change, status):
    assert lib.rt_attention(None, *{**ATTENTION, **change}.values()) == status, lib.rt_last_error()


CACHE = dict(k=0x1000, v=0x2000, table=0x3000, lens=0x4000, pages=50, kv_heads=2, page_len=16, head_dim=64, seqs=3, table_len=20)


def cache(**change):
    c = {**CACHE, **change}
    return _lib.PagedKV(*(c[n] for n, _ in _lib.PagedKV._fields_))


BAD_CACHES = [({"pages": 0}, SHAPE), ({"kv_heads": 0}, SHAPE), ({"page_len": 0}, SHAPE), ({"head_dim": 0}, SHAPE), ({"seqs": 0}, SHAPE), ({"table_len": 0}, SHAPE),
              ({"seqs": 70000}, SIZE), ({"table_len": 1 << 30}, SIZE), ({"pages": 1 << 31}, SIZE), ({"page_len": 1 << 31}, SIZE), ({"pages": 1 << 30, "page_len": 1 << 20}, SIZE),
              ({"k": None}, NULL), ({"v": None}, NULL), ({"table": None}, NULL), ({"lens": None}, NULL),
              ({"k": 0x1001}, ALIGN), ({"v": 0x1001}, ALIGN), ({"table": 0x1002}, ALIGN), ({"lens": 0x1002}, ALIGN)]


def append(lib, kv, **change):
    a = {**dict(elem_bytes=2, kv=kv, starts=SOME, tokens=5, k=SOME, k_strides=None, v=SOME, v_strides=None), **change}
    return lib.rt_paged_append(None, *a.values())


def attend(lib, kv, **change):
    a = {**dict(dt=_lib.F16, q=SOME, q_strides=None, tokens=5, heads=8, kv=kv, starts=SOME, y=SOME, lse=None, weights=None, weights_out=None, scale=0.1, window=0, sinks=0), **change}
    return lib.rt_paged_attention(None, *a.values())


def evict(lib, kv, **change):
    a = {**dict(elem_bytes=2, kv=kv, weights=SOME, keep=40, first=4, recent=10, table_out=SOME, lens_out=SOME, weights_out=SOME), **change}
    return lib.rt_paged_evict(None, *a.values())


@pytest.mark.parametrize("call", [append, attend, evict])
@pytest.mark.parametrize("change, status", BAD_CACHES)
def test_caches(lib, call, change, status):
    got = call(lib, cache(**change))
    assert got == status, lib.rt_last_error()
    assert call(lib, None) == NULL


@pytest.mark.parametrize("call, change, status", [
    (append, {}, OK_BUT_NO_DEVICE), (append, {"elem_bytes": 1}, ARG), (append, {"tokens": 0}, SHAPE), (append, {"tokens": 1 << 31}, SIZE), (append, {"k": None}, NULL),
    (append, {"v": None}, NULL), (append, {"starts": None}, NULL), (append, {"k": ODD}, ALIGN), (append, {"v": ODD}, ALIGN), (append, {"starts": ctypes.c_void_p(0x1002)}, ALIGN),
    (append, {"k_strides": s(1 << 40, 64)}, SIZE), (append, {"v_strides": s(64, 1 << 40)}, SIZE), (append, {"k_strides": s(0, 0)}, OK_BUT_NO_DEVICE),
    (attend, {}, OK_BUT_NO_DEVICE), (attend, {"dt": _lib.U32}, DTYPE), (attend, {"tokens": 0}, SHAPE), (attend, {"heads": 0}, SHAPE), (attend, {"heads": 7}, SHAPE),
    (attend, {"q": None}, NULL), (attend, {"y": None}, NULL), (attend, {"starts": None}, NULL), (attend, {"q": ODD}, ALIGN), (attend, {"y": ODD}, ALIGN),
    (attend, {"lse": ctypes.c_void_p(0x1002)}, ALIGN), (attend, {"weights": SOME}, NULL), (attend, {"weights_out": SOME}, NULL),
    (attend, {"weights": SOME, "weights_out": SOME}, OK_BUT_NO_DEVICE), (attend, {"weights": SOME, "weights_out": ctypes.c_void_p(0x1002)}, ALIGN), (attend, {"scale": float("nan")}, ARG),
    (attend, {"q_strides": s(1 << 40, 64)}, SIZE),
    (evict, {}, OK_BUT_NO_DEVICE), (evict, {"elem_bytes": 8}, ARG), (evict, {"keep": 0}, ARG), (evict, {"keep": 321}, ARG), (evict, {"keep": 320}, OK_BUT_NO_DEVICE),
    (evict, {"first": 31}, ARG), (evict, {"first": 30}, OK_BUT_NO_DEVICE), (evict, {"first": (1 << 32) - 1, "recent": 2}, ARG), (evict, {"weights": None}, NULL),
    (evict, {"table_out": None}, NULL), (evict, {"lens_out": None}, NULL), (evict, {"weights_out": None}, NULL), (evict, {"weights_out": ctypes.c_void_p(0x1002)}, ALIGN),
])
def test_calls(lib, call, change, status):
    assert call(lib, cache(), **change) == status, lib.rt_last_error()


def test_head_dims_of_paged_attention(lib):
    assert attend(lib, cache(head_dim=513)) == SIZE
    assert append(lib, cache(head_dim=513)) == OK_BUT_NO_DEVICE                # moving rows has no such limit


# sequences x KV heads x keys of 65535 x 65535 x 2^20: no weights can have as many elements, and the sizes that go by them would not fit 64 bits
WIDE = dict(seqs=65535, kv_heads=65535, page_len=1, pages=1, head_dim=8, table_len=1 << 20)


def test_sizes_that_pass_64_bits(lib):
    assert attend(lib, cache(**WIDE), heads=65535, weights=SOME, weights_out=SOME) == SIZE
    assert attend(lib, cache(**WIDE), heads=65535) == OK_BUT_NO_DEVICE
    assert evict(lib, cache(**WIDE)) == SIZE
    assert attend(lib, cache(), q_strides=s(0, 0), tokens=1 << 30, heads=1 << 31) == SIZE
    assert attend(lib, cache(), q_strides=s(0, 0), tokens=1 << 20, heads=1 << 10) == OK_BUT_NO_DEVICE


class Shape:
    """stands for a buffer: the Python layer looks at its shape and type first"""

    def __init__(self, shape, dt, numel=None):
        self.shape, self.dt, self.ptr = shape, dt, ctypes.c_void_p(0x1000)
        self.numel = numel if numel is not None else int(__import__("math").prod(shape))


def test_python_layer():
    from ratchet_amd.runtime import Device, PagedCache

    dev = Device.__new__(Device)
    dev.lib, dev.handle = _lib.load(), None
    q, k = Shape((1, 4, 8, 64), _lib.F16), Shape((1, 2, 20, 64), _lib.F16)
    for bad in (dict(k=Shape((1, 2, 20, 64), _lib.BF16)), dict(v=Shape((1, 2, 21, 64), _lib.F16)), dict(lens=Shape((2,), _lib.I32)), dict(lens=Shape((1,), _lib.F32)),
                dict(q_strides=(0, 64, 257, 1)), dict(q_strides=(0, -1, 64, 1)), dict(out=Shape((1, 4, 8, 64), _lib.F32)), dict(lse=Shape((1, 4, 9), _lib.F32))):
        with pytest.raises(ValueError):
            dev.attention(**{**dict(q=q, k=k, v=k, out=q), **bad})
    table, lens, pages = Shape((3, 5), _lib.I32), Shape((3,), _lib.I32), Shape((9, 2, 16, 64), _lib.F16)
    for bad in ((pages, Shape((9, 2, 16, 32), _lib.F16), table, lens), (pages, pages, Shape((3, 5), _lib.F32), lens), (pages, pages, table, Shape((4,), _lib.I32))):
        with pytest.raises(ValueError):
            PagedCache(*bad)
    cache = PagedCache(pages, pages, table, lens)
    rows, starts, w = Shape((6, 2, 64), _lib.F16), Shape((4,), _lib.I32), Shape((3, 2, 80), _lib.F32)
    for bad in (dict(k=Shape((6, 3, 64), _lib.F16)), dict(v=Shape((6, 2, 64), _lib.F32)), dict(starts=Shape((3,), _lib.I32)), dict(k_strides=(129, 64))):
        with pytest.raises(ValueError):
            dev.paged_append(cache, **{**dict(starts=starts, k=rows, v=rows), **bad})
    q = Shape((6, 4, 64), _lib.F16)
    for bad in (dict(q=Shape((6, 4, 32), _lib.F16)), dict(starts=Shape((4,), _lib.U32)), dict(weights=Shape((3, 2, 79), _lib.F32)), dict(weights_out=w), dict(q_strides=(257, 64)),
                dict(out=Shape((6, 4, 63), _lib.F16))):
        with pytest.raises(ValueError):
            dev.paged_attention(cache=cache, **{**dict(q=q, starts=starts, out=q), **bad})
    for bad in (dict(weights=Shape((3, 2, 81), _lib.F32)), dict(to=Shape((3, 6), _lib.I32)), dict(lens_out=Shape((2,), _lib.I32)), dict(weights_out=Shape((3, 2, 80), _lib.I32))):
        with pytest.raises(ValueError):
            dev.paged_evict(cache, **{**dict(weights=w, keep=10), **bad})
