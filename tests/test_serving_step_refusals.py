"""What rotary positions of tokens, attention with changed scores and sampling refuse, before any HIP call; and what the Python layer refuses.  No GPU needed."""
import ctypes
import math

import numpy as np
import pytest

from ratchet_amd import _lib, rope_divisors
from ratchet_amd.runtime import Device, PagedCache

SOME, ODD, OTHER = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001), ctypes.c_void_p(0x9000)
HALF = ctypes.c_void_p(0x1002)
FINE, NULL, DTYPE, SHAPE, SIZE, ARG, ALIGN = 8, 1, 2, 4, 6, 7, 9                     # FINE: there is no device, which is found last
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def u4(*v):
    return (ctypes.c_uint32 * 4)(*v)


def s(*v):
    return (ctypes.c_uint64 * len(v))(*v)


ROPE = dict(dt=_lib.F16, x=SOME, x_strides=None, y=OTHER, y_strides=None, tokens=10, heads=8, head_dim=64, positions=SOME, turns=SOME, dim=64, factor=1.0, interleaved=0)
TABLES = [({"dt": _lib.I32}, DTYPE), ({"dim": 0}, SHAPE), ({"dim": 7}, SHAPE), ({"dim": 66}, SHAPE), ({"factor": NAN}, ARG), ({"factor": INF}, ARG), ({"factor": 0.0}, FINE),
          ({"interleaved": 2}, ARG), ({"interleaved": 1}, FINE), ({"turns": None}, NULL), ({"turns": ctypes.c_void_p(0x1004)}, ALIGN)]


@pytest.mark.parametrize("change, status", TABLES + [
    ({}, FINE), ({"x": None}, NULL), ({"y": None}, NULL), ({"positions": None}, NULL), ({"x": ODD}, ALIGN), ({"y": ODD}, ALIGN), ({"positions": HALF}, ALIGN),
    ({"tokens": 0}, SHAPE), ({"heads": 0}, SHAPE), ({"head_dim": 0}, SHAPE), ({"heads": 70000}, SIZE), ({"tokens": 1 << 31}, SIZE), ({"head_dim": 1 << 17}, SIZE),
    ({"head_dim": 2048, "dim": 1026}, SIZE), ({"head_dim": 2048, "dim": 1024}, FINE),
    ({"x_strides": s(0, 0)}, FINE), ({"y_strides": s(0, 64)}, ARG), ({"y_strides": s(512, 63)}, ARG), ({"y_strides": s(511, 64)}, ARG), ({"y_strides": s(64, 640)}, FINE),
    ({"y_strides": s(64, 639)}, ARG), ({"x_strides": s(1 << 41, 64)}, SIZE), ({"x_strides": s((1 << 64) - 1, 64)}, SIZE), ({"y": SOME}, FINE),
    ({"y": SOME, "y_strides": s(1024, 64)}, ARG), ({"y": SOME, "y_strides": s(1024, 64), "x_strides": s(1024, 64)}, FINE),
])
def test_rope_tokens(lib, change, status):
    assert lib.rt_rope_tokens(None, *{**ROPE, **change}.values()) == status, lib.rt_last_error()


CACHE = dict(k=0x1000, v=0x2000, table=0x3000, lens=0x4000, pages=50, kv_heads=2, page_len=16, head_dim=64, seqs=3, table_len=20)


def cache(**change):
    c = {**CACHE, **change}
    return _lib.PagedKV(*(c[n] for n, _ in _lib.PagedKV._fields_))


BAD_CACHES = [({"pages": 0}, SHAPE), ({"kv_heads": 0}, SHAPE), ({"page_len": 0}, SHAPE), ({"seqs": 0}, SHAPE), ({"table_len": 0}, SHAPE), ({"seqs": 70000}, SIZE),
              ({"table_len": 1 << 30}, SIZE), ({"k": None}, NULL), ({"lens": None}, NULL), ({"v": 0x1001}, ALIGN), ({"table": 0x1002}, ALIGN)]
APPEND = dict(dt=_lib.F16, kv=cache(), starts=SOME, tokens=10, q=SOME, q_strides=None, heads=8, y=OTHER, y_strides=None, k=SOME, k_strides=None, v=SOME, v_strides=None, turns=SOME,
              dim=64, factor=1.0, interleaved=0)


@pytest.mark.parametrize("change, status", TABLES + [({"kv": cache(**c)}, r) for c, r in BAD_CACHES] + [
    ({}, FINE), ({"kv": None}, NULL), ({"starts": None}, NULL), ({"q": None}, NULL), ({"y": None}, NULL), ({"k": None}, NULL), ({"v": None}, NULL),
    ({"starts": HALF}, ALIGN), ({"q": ODD}, ALIGN), ({"y": ODD}, ALIGN), ({"k": ODD}, ALIGN), ({"v": ODD}, ALIGN),
    ({"tokens": 0}, SHAPE), ({"heads": 0}, SHAPE), ({"heads": 70000}, SIZE), ({"tokens": 1 << 31}, SIZE), ({"q_strides": s(1 << 41, 64)}, SIZE), ({"k_strides": s(1 << 41, 64)}, SIZE),
    ({"v_strides": s(1 << 41, 64)}, SIZE), ({"y_strides": s(512, 1)}, ARG), ({"y": SOME}, FINE), ({"y": SOME, "q_strides": s(1024, 64)}, ARG), ({"heads": 3}, FINE),
])
def test_paged_rope_append(lib, change, status):
    assert lib.rt_paged_rope_append(None, *{**APPEND, **change}.values()) == status, lib.rt_last_error()


def test_rope_turns(lib):
    turns = np.zeros(4, np.uint64)
    put = turns.ctypes.data
    good = np.array([1.0, 2.0, 0.01, 1e30])
    assert lib.rt_rope_turns(8, 10000.0, good.ctypes.data, put) == 0
    assert lib.rt_rope_turns(8, 10000.0, None, None) == NULL
    assert lib.rt_rope_turns(0, 10000.0, None, put) == SHAPE and lib.rt_rope_turns(7, 10000.0, None, put) == SHAPE
    for base in (0.0, -1.0, NAN, INF):
        assert lib.rt_rope_turns(8, base, None, put) == ARG
    for bad in (0.0, -1.0, NAN, INF):
        divisors = np.array([1.0, 1.0, 1.0, bad])
        assert lib.rt_rope_turns(8, 10000.0, divisors.ctypes.data, put) == ARG


@pytest.mark.parametrize("base, divisors", [(10000.0, None), (500000.0, 32.0), (10000.0, 0.01), (0.5, None)])
def test_rope_turns_are_fractions_of_a_turn(lib, base, divisors):
    """to the last of 64 bits, but what long double loses: 2^-64 of the frequency and 2^-64 of a turn"""
    from fractions import Fraction

    dim = 96
    turns, d = np.zeros(dim // 2, np.uint64), None if divisors is None else np.full(dim // 2, divisors)
    assert lib.rt_rope_turns(dim, base, None if d is None else d.ctypes.data, turns.ctypes.data) == 0
    two_pi = Fraction(2 * 31415926535897932384626433832795028841971, 10 ** 40)
    for i in range(dim // 2):
        # base^(-2i / dim) from its (dim / 2)th power: compared as (turns * 2 pi * divisor)^(dim / 2) = base^-i where nothing has wrapped
        f = (np.longdouble(base) ** (-np.longdouble(2 * i) / dim)) / np.longdouble(divisors or 1.0)
        hi = float(f)
        exact = (Fraction(hi) + Fraction(float(f - np.longdouble(hi)))) / two_pi
        off = abs((Fraction(int(turns[i]), 2 ** 64) - exact + Fraction(1, 2)) % 1 - Fraction(1, 2))
        assert off <= (2 + 8 * exact) / 2 ** 64, (i, float(off * 2 ** 64))


def test_rope_divisors():
    d = rope_divisors(64, 10000.0, 8.0, 4096, low=1.0, high=4.0)
    turns = 4096 * 10000.0 ** (-np.arange(32) / 32) / (2 * np.pi)
    assert (d[turns >= 4] == 1).all() and (d[turns <= 1] == 8).all() and ((d > 1) & (d < 8))[(turns > 1) & (turns < 4)].all()


def scores(cap=0.0, slopes=None, documents=None, n=0, prefix=None):
    return ctypes.byref(_lib.Scores(cap, slopes, documents, n, prefix))


ATTENTION = dict(dt=_lib.F16, q=SOME, q_shape=u4(2, 8, 16, 64), q_strides=None, k=SOME, k_strides=None, v=SOME, v_strides=None, kv_shape=u4(2, 2, 100, 64), lens=None, y=SOME,
                 y_strides=None, lse=None, scale=0.125, causal=1, window=0, sinks=0, scores=scores(cap=30.0))
SCORES = [({"scores": scores()}, FINE), ({"scores": None}, NULL), ({"scores": scores(cap=-1.0)}, ARG), ({"scores": scores(cap=NAN)}, ARG), ({"scores": scores(cap=INF)}, ARG),
          ({"scores": scores(cap=3.3e38)}, ARG), ({"scores": scores(cap=1e-45)}, ARG), ({"scores": scores(slopes=0x1000)}, FINE), ({"scores": scores(slopes=0x1002)}, ALIGN),
          ({"scores": scores(prefix=0x1000)}, FINE), ({"scores": scores(prefix=0x1002)}, ALIGN), ({"scores": scores(n=3)}, SHAPE)]


@pytest.mark.parametrize("change, status", SCORES + [
    ({}, FINE), ({"q": None}, NULL), ({"dt": _lib.U32}, DTYPE), ({"q_shape": None}, NULL), ({"kv_shape": u4(2, 3, 100, 64)}, SHAPE), ({"y": ODD}, ALIGN),
    ({"scores": scores(documents=0x1000, n=5)}, FINE), ({"scores": scores(documents=0x1002, n=5)}, ALIGN), ({"scores": scores(documents=0x1000)}, SHAPE),
    ({"scores": scores(documents=0x1000, n=1 << 31)}, SIZE), ({"scores": scores(documents=0x1000, n=5, prefix=0x1000)}, FINE),
    ({"causal": 0, "scores": scores(prefix=0x1000)}, ARG), ({"causal": 0, "scores": scores(documents=0x1000, n=5)}, FINE), ({"causal": 0, "window": 4}, ARG),
])
def test_attention_scored(lib, change, status):
    assert lib.rt_attention_scored(None, *{**ATTENTION, **change}.values()) == status, lib.rt_last_error()


PAGED = dict(dt=_lib.F16, q=SOME, q_strides=None, tokens=10, heads=8, kv=cache(), starts=SOME, y=SOME, lse=None, scale=0.125, window=0, sinks=0, scores=scores(cap=30.0))


@pytest.mark.parametrize("change, status", SCORES + [({"kv": cache(**c)}, r) for c, r in BAD_CACHES] + [
    ({}, FINE), ({"q": None}, NULL), ({"kv": None}, NULL), ({"starts": None}, NULL), ({"heads": 5}, SHAPE), ({"tokens": 0}, SHAPE), ({"scores": scores(documents=0x1000, n=5)}, ARG),
])
def test_paged_attention_scored(lib, change, status):
    assert lib.rt_paged_attention_scored(None, *{**PAGED, **change}.values()) == status, lib.rt_last_error()


SAMPLE = dict(dt=_lib.F32, x=SOME, row_stride=1000, rows=4, vocab=1000, temperature=SOME, top_k=SOME, top_p=SOME, min_p=SOME, uniform=SOME, tokens=SOME, probs=SOME)


@pytest.mark.parametrize("change, status", [
    ({}, FINE), ({"dt": _lib.I32}, DTYPE), ({"rows": 0}, SHAPE), ({"vocab": 0}, SHAPE), ({"vocab": (1 << 24) + 1}, SIZE), ({"vocab": 1 << 24}, FINE), ({"rows": 1 << 22}, SIZE),
    ({"row_stride": 1 << 60}, SIZE), ({"row_stride": 0}, FINE), ({"x": None}, NULL), ({"uniform": None}, NULL), ({"tokens": None}, NULL),
    ({"temperature": None, "top_k": None, "top_p": None, "min_p": None, "probs": None}, FINE), ({"x": HALF}, ALIGN), ({"x": HALF, "dt": _lib.F16}, FINE)] + [
    ({name: HALF}, ALIGN) for name in ("temperature", "top_k", "top_p", "min_p", "uniform", "tokens", "probs")])
def test_sample(lib, change, status):
    assert lib.rt_sample(None, *{**SAMPLE, **change}.values()) == status, lib.rt_last_error()


class Shape:
    """stands for a buffer: its shape and type are what is looked at"""

    def __init__(self, shape, dt):
        self.shape, self.dt, self.ptr, self.numel = shape, dt, ctypes.c_void_p(0x1000), math.prod(shape)


class Library:
    """stands for the library: the names of the calls that reach it"""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0
        return call


@pytest.fixture
def dev():
    d = Device.__new__(Device)
    d.lib, d.handle = Library(), None
    yield d
    d.handle = None


F16, F32, I32, U32 = _lib.F16, _lib.F32, _lib.I32, _lib.U32
PAGES = PagedCache(Shape((9, 2, 16, 64), F16), Shape((9, 2, 16, 64), F16), Shape((3, 5), I32), Shape((3,), I32))
X, Q, K = Shape((6, 4, 64), F16), Shape((1, 4, 8, 64), F16), Shape((1, 2, 20, 64), F16)
NEW, STARTS, TABLE = Shape((6, 2, 64), F16), Shape((4,), I32), Shape((32, 2), U32)


@pytest.mark.parametrize("call", [
    lambda d: d.rope_tokens(Shape((6, 64), F16), Shape((6,), I32), TABLE), lambda d: d.rope_tokens(X, Shape((5,), I32), TABLE), lambda d: d.rope_tokens(X, Shape((6,), U32), TABLE),
    lambda d: d.rope_tokens(X, Shape((6,), I32), Shape((32, 2), I32), out=X), lambda d: d.rope_tokens(X, Shape((6,), I32), Shape((64,), U32), out=X),
    lambda d: d.rope_tokens(X, Shape((6,), I32), TABLE, out=Shape((6, 4, 32), F16)), lambda d: d.rope_tokens(X, Shape((6,), I32), TABLE, out=Shape((6, 4, 64), F32)),
    lambda d: d.rope_tokens(X, Shape((6,), I32), TABLE, strides=(256,), out=X), lambda d: d.rope_tokens(X, Shape((6,), I32), TABLE, strides=(257, 64), out=X),
    lambda d: d.rope_tokens(X, Shape((6,), I32), TABLE, strides=(-256, 64), out=X), lambda d: d.rope_tokens(X, Shape((6,), I32), TABLE, out=X, out_strides=(256, 65)),
    lambda d: d.rope_table(-2), lambda d: d.rope_table(64, divisors=[1.0, 2.0]),
    lambda d: d.paged_rope_append(PAGES, STARTS, X, NEW, Shape((6, 2, 32), F16), TABLE), lambda d: d.paged_rope_append(PAGES, STARTS, Shape((5, 4, 64), F16), NEW, NEW, TABLE),
    lambda d: d.paged_rope_append(PAGES, STARTS, Shape((6, 4, 64), F32), NEW, NEW, TABLE), lambda d: d.paged_rope_append(PAGES, Shape((3,), I32), X, NEW, NEW, TABLE),
    lambda d: d.paged_rope_append(PAGES, STARTS, X, NEW, NEW, Shape((32, 3), U32)), lambda d: d.paged_rope_append(PAGES, STARTS, X, NEW, NEW, TABLE, out=Shape((6, 4, 64), F32)),
    lambda d: d.paged_rope_append(PAGES, STARTS, X, NEW, NEW, TABLE, out=X, k_strides=(129, 64)),
    lambda d: d.attention(Q, K, K, out=Q, slopes=Shape((3,), F32)), lambda d: d.attention(Q, K, K, out=Q, slopes=Shape((4,), F16)), lambda d: d.attention(Q, K, K, out=Q, documents=Shape((2, 5), I32)),
    lambda d: d.attention(Q, K, K, out=Q, documents=Shape((1, 1), I32)), lambda d: d.attention(Q, K, K, out=Q, documents=Shape((1, 4), F32)),
    lambda d: d.attention(Q, K, K, out=Q, prefix=Shape((2,), I32)), lambda d: d.attention(Q, K, K, out=Q, documents=Shape((1, 4), I32), prefix=Shape((1,), I32)),
    lambda d: d.attention(Q, K, K, out=Q, documents=Shape((1, 4), I32), prefix=Shape((1, 4), I32)),
    lambda d: d.paged_attention(X, PAGES, STARTS, out=X, slopes=Shape((2,), F32)), lambda d: d.paged_attention(X, PAGES, STARTS, out=X, prefix=Shape((4,), I32)),
    lambda d: d.paged_attention(X, PAGES, STARTS, out=X, cap=5.0, weights=Shape(PAGES.weights_shape, F32)),
    lambda d: d.sample(Shape((4, 5, 6), F32), Shape((4,), F32)), lambda d: d.sample(Shape((4, 6), F32), Shape((5,), F32)), lambda d: d.sample(Shape((4, 6), F32), Shape((4,), I32)),
    lambda d: d.sample(Shape((4, 6), F32), Shape((4,), F32), top_k=Shape((4,), F32)), lambda d: d.sample(Shape((4, 6), F32), Shape((4,), F32), temperature=Shape((1,), F32)),
    lambda d: d.sample(Shape((4, 6), F32), Shape((4,), F32), out=Shape((4,), F32)), lambda d: d.sample(Shape((4, 6), F32), Shape((4,), F32), probs=Shape((4,), I32), out=Shape((4,), I32)),
    lambda d: d.sample(Shape((4, 6), F32), Shape((4,), F32), out=Shape((4,), I32), row_stride=7),
])
def test_python_refuses(dev, call):
    with pytest.raises(ValueError):
        call(dev)
    assert dev.lib.calls == []


def test_python_passes_on_what_is_right(dev):
    dev.rope_tokens(X, Shape((6,), I32), TABLE, out=X)
    dev.paged_rope_append(PAGES, STARTS, X, NEW, NEW, TABLE, out=X)
    dev.attention(Q, K, K, out=Q, documents=Shape((1, 4), I32), prefix=Shape((1, 3), I32), slopes=Shape((4,), F32), cap=3.0)
    dev.attention(Q, K, K, out=Q)
    dev.paged_attention(X, PAGES, STARTS, out=X, cap=3.0, prefix=Shape((3,), I32))
    dev.sample(Shape((4, 6), F32), Shape((4,), F32), out=Shape((4,), I32))
    assert dev.lib.calls == ["rt_rope_tokens", "rt_paged_rope_append", "rt_attention_scored", "rt_attention", "rt_paged_attention_scored", "rt_sample"]
