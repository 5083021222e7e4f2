"""Rotary positions of tokens, alone and into the paged cache, against complex rotations in long double.

Bound (u = 2^-24): the angle, less than an eighth of a turn of it, is rounded as a float and times 2 pi, 2u of at most 0.79 in all; the series' terms add less than 1.2u of 1;
the factor rounds once more: a sine or cosine is off by less than 4u, times |factor|.  Each of two products takes that and a rounding, their sum one more:
6u |factor| (|x1| + |x2|), and what is stored is rounded to the type (half a step)."""
import ctypes

import numpy as np
import pytest

import attention_ref as ref
from attention_ref import HALF_STEP, TINY, U
from ratchet_amd import _lib, rope_divisors
from ratchet_amd._lib import check

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def dev():
    from ratchet_amd import Device

    d = Device(0)
    yield d
    d.close()


def turned(x, positions, dim, base, divisors, factor, interleaved, dtype):
    """the rotated rows and their bounds"""
    half = dim // 2
    f = np.longdouble(base) ** (-2 * np.arange(half).astype(np.longdouble) / dim) / (1.0 if divisors is None else np.asarray(divisors))
    angle = np.asarray(positions).astype(np.longdouble)[:, None] * f
    cos, sin = np.cos(angle).astype(np.float64)[:, None] * factor, np.sin(angle).astype(np.float64)[:, None] * factor
    one, two = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, half), slice(half, dim))
    y, off = x.copy(), np.zeros_like(x)
    y[..., one], y[..., two] = x[..., one] * cos - x[..., two] * sin, x[..., one] * sin + x[..., two] * cos
    both = 6 * U * abs(factor) * (np.abs(x[..., one]) + np.abs(x[..., two]))
    off[..., one] = off[..., two] = both
    off[..., :dim] += HALF_STEP[dtype] * (np.abs(y[..., :dim]) + off[..., :dim]) + TINY[dtype]
    return y, off


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, heads, head_dim, dim", [(1, 1, 2, 2), (1, 40, 128, 128), (64, 40, 128, 128), (7, 3, 80, 32), (5, 2, 96, 96), (9, 5, 64, 48), (3, 4, 20, 10), (17, 3, 7, 6),
                                                          (2, 2, 256, 64), (3, 1, 1024, 1024), (300, 6, 40, 16), (2, 3, 24, 8), (33, 130, 64, 64), (4, 2, 72, 24),
                                                          # several tokens to a block, the last one's fewer
                                                          (1500, 1, 64, 64), (2001, 2, 96, 32), (1111, 3, 20, 8), (70001, 1, 2, 2), (3001, 1, 7, 6), (1300, 5, 40, 40), (515, 1, 1024, 1024),
                                                          (6000, 1, 128, 128)])
def test_shapes(dev, dtype, interleaved, tokens, heads, head_dim, dim):
    rng = np.random.default_rng(tokens + head_dim + dim)
    x, positions = ref.rounded(rng.standard_normal((tokens, heads, head_dim)), dtype), rng.integers(0, 5000, tokens).astype(np.int32)
    want, off = turned(x, positions, dim, 10000.0, None, 1.0, interleaved, dtype)
    table, at = dev.rope_table(dim), dev.upload(positions)
    out = dev.rope_tokens(ref.upload(dev, x, dtype), at, table, interleaved=interleaved)
    ref.check(ref.values(out.to_numpy(), dtype), want, off, "out of place")
    here = ref.upload(dev, x, dtype)
    dev.rope_tokens(here, at, table, interleaved=interleaved, out=here)
    assert np.array_equal(here.to_numpy(), out.to_numpy())      # in place


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_and_negative_positions(dev, dtype, interleaved):
    rng = np.random.default_rng(0)
    positions = np.array([0, 1, -1, 131071, 2 ** 20, -2 ** 20, 2 ** 31 - 1, -2 ** 31, 12345678, 4096], np.int32)
    x = ref.rounded(rng.standard_normal((len(positions), 4, 64)), dtype)
    want, off = turned(x, positions, 64, 500000.0, None, 1.0, interleaved, dtype)
    out = dev.rope_tokens(ref.upload(dev, x, dtype), dev.upload(positions), dev.rope_table(64, 500000.0), interleaved=interleaved)
    ref.check(ref.values(out.to_numpy(), dtype), want, off, "far")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("factor", [1.0, 1.3465735902799727, -0.5, 0.0])
def test_scaled_tables(dev, dtype, factor):
    rng = np.random.default_rng(1)
    positions = rng.integers(0, 10 ** 6, 50).astype(np.int32)
    x = ref.rounded(rng.standard_normal((50, 4, 96)), dtype)
    own = 1 + 40 * rng.random(48)
    by_waves = rope_divisors(96, 10000.0, 32.0, 4096)
    assert by_waves[0] == 1 and by_waves[-1] == 32 and (np.diff(by_waves) >= 0).all()
    factor = float(np.float32(factor))
    for divisors in (8.0, own, by_waves, 0.25):
        want, off = turned(x, positions, 96, 10000.0, np.broadcast_to(divisors, 48), factor, False, dtype)
        out = dev.rope_tokens(ref.upload(dev, x, dtype), dev.upload(positions), dev.rope_table(96, 10000.0, divisors), factor=factor)
        ref.check(ref.values(out.to_numpy(), dtype), want, off, "scaled")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 2, 8])
def test_windows_of_a_projection(dev, dtype, interleaved, shift):
    """rows with strides and off the vector grid; what lies between them stays as it was"""
    rng = np.random.default_rng(shift)
    n, heads, kv_heads, d = 21, 6, 2, 32
    w = (heads + 2 * kv_heads) * d + shift
    whole = ref.rounded(rng.standard_normal(shift + n * w), dtype)
    positions = rng.integers(0, 9999, n).astype(np.int32)
    buf = ref.upload(dev, whole, dtype)
    rows = whole[shift:].reshape(n, w)
    x = rows[:, :(heads + kv_heads) * d].reshape(n, heads + kv_heads, d)
    want, off = turned(x, positions, 16, 10000.0, None, 1.0, interleaved, dtype)
    view = buf.view(shift, x.shape)
    table, at = dev.rope_table(16), dev.upload(positions)
    out = dev.rope_tokens(view, at, table, interleaved=interleaved, strides=(w, d))
    ref.check(ref.values(out.to_numpy(), dtype), want, off, "windows")
    # head by head in memory, a gap of three behind each
    apart = ref.upload(dev, np.full((heads + kv_heads) * n * (d + 3), 7.0), dtype)
    dev.rope_tokens(view, at, table, interleaved=interleaved, strides=(w, d), out=apart.view(0, x.shape), out_strides=(d + 3, n * (d + 3)))
    there = apart.to_numpy().reshape(heads + kv_heads, n, d + 3)
    assert np.array_equal(there[:, :, :d].transpose(1, 0, 2), out.to_numpy()) and (ref.values(there[:, :, d:], dtype) == 7).all()
    dev.rope_tokens(view, at, table, interleaved=interleaved, strides=(w, d), out=view, out_strides=(w, d))
    after = buf.to_numpy()
    assert np.array_equal(after[shift:].reshape(n, w)[:, :x[0].size].reshape(x.shape), out.to_numpy())
    assert np.array_equal(ref.values(after[shift:].reshape(n, w)[:, x[0].size:], dtype), rows[:, x[0].size:])


def test_many_tokens(dev):
    """more tokens than a row of the grid has blocks"""
    n, d = (1 << 22) + 1001, 2
    x = np.random.default_rng(3).standard_normal((n, 1, d)).astype(np.float32)
    positions = (np.arange(n) % 5000).astype(np.int32)
    out = dev.rope_tokens(dev.upload(x), dev.upload(positions), dev.rope_table(2)).to_numpy()
    for s in (slice(0, 1000), slice(n - 2000, n)):
        want, off = turned(x[s].astype(np.float64), positions[s], 2, 10000.0, None, 1.0, False, "f32")
        ref.check(out[s], want, off, "many")


def test_many_tokens_of_many_heads(dev):
    """a token to a block, more than a row of the grid has; all tokens are one row, 2.2 GB of results"""
    n, heads = (1 << 22) + 1001, 130
    x = np.random.default_rng(4).standard_normal((1, heads, 2)).astype(np.float16)
    positions = (np.arange(n) % 5000).astype(np.int32)
    row, at, table, out = dev.upload(x), dev.upload(positions), dev.rope_table(2), dev.empty((n, heads, 2), _lib.F16)
    strides = (ctypes.c_uint64 * 2)(0, 2)
    check(dev.lib.rt_rope_tokens(dev.handle, _lib.F16, row.ptr, strides, out.ptr, None, n, heads, 2, at.ptr, table.ptr, 2, 1.0, 0))
    for first in (0, (1 << 22) - 500, n - 1000):
        got = out.view(first * heads * 2, (1000, heads, 2)).to_numpy()
        want, off = turned(np.repeat(x.astype(np.float64), 1000, axis=0), positions[first:first + 1000], 2, 10000.0, None, 1.0, False, "f16")
        ref.check(ref.values(got, "f16"), want, off, "many")


def into_the_cache(dev, rng, dtype, interleaved, heads, kv_heads, d, dim, page, lens, new, hole):
    p = ref.Paged(rng, dtype, heads, kv_heads, d, page, lens, new, holes=[hole], spare=0)
    p.lens[1] = p.cap + 3
    k, v = (ref.rounded(rng.standard_normal((p.tokens, kv_heads, d)), dtype) for _ in range(2))
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    at = np.concatenate([p.lens[b] - p.new[b] + np.arange(p.new[b]) for b in range(len(p.lens))])
    # two rows in front of the first sequence and three behind the last belong to nobody
    starts = p.starts + 2
    pad = lambda x: np.concatenate([np.full((2,) + x.shape[1:], np.nan), x, np.full((3,) + x.shape[1:], np.nan)])        # noqa: E731
    q = pad(p.q)
    kept = ref.upload(dev, np.full(q.shape, 5.0), dtype)
    out = dev.paged_rope_append(cache, dev.upload(starts), ref.upload(dev, q, dtype), ref.upload(dev, pad(k), dtype), ref.upload(dev, pad(v), dtype), dev.rope_table(dim), factor=1.25,
                                interleaved=interleaved, out=kept)
    got = ref.values(out.to_numpy(), dtype)
    assert (got[:2] == 5).all() and (got[-3:] == 5).all()
    want, off = turned(p.q, at, dim, 10000.0, None, 1.25, interleaved, dtype)
    ref.check(got[2:-3], want, off, "q")
    turned_k, off_k = turned(k, at, dim, 10000.0, None, 1.25, interleaved, dtype)
    k_off = np.zeros_like(p.k)
    for b in range(len(p.lens)):
        for j in range(p.starts[b], p.starts[b + 1]):
            t = max(int(p.lens[b]), 0) - int(p.starts[b + 1] - j)
            if 0 <= t < p.cap and 0 <= p.table[b, t // page] < p.pages:
                where = p.table[b, t // page], slice(None), t % page
                p.k[where], k_off[where], p.v[where] = turned_k[j], off_k[j], v[j]
    ref.check(ref.values(cache.k_pages.to_numpy(), dtype), p.k, k_off, "k")
    assert np.array_equal(ref.values(cache.v_pages.to_numpy(), dtype), p.v)
    # q in place: the same
    here = ref.upload(dev, q, dtype)
    dev.paged_rope_append(cache, dev.upload(starts), here, ref.upload(dev, pad(k), dtype), ref.upload(dev, pad(v), dtype), dev.rope_table(dim), factor=1.25, interleaved=interleaved, out=here)
    assert np.array_equal(ref.values(here.to_numpy(), dtype)[2:-3], got[2:-3]) and np.isnan(ref.values(here.to_numpy(), dtype)[:2]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads, kv_heads, d, dim", [(4, 2, 64, 64), (3, 1, 20, 8), (8, 8, 80, 32), (2, 2, 7, 6), (40, 8, 128, 128)])
@pytest.mark.parametrize("page", [16, 7, 1])
def test_into_the_cache(dev, dtype, interleaved, heads, kv_heads, d, dim, page):
    # a first token, a prompt, a later piece, nothing, a page that is missing, more new tokens than lens counts, tokens beyond the table
    into_the_cache(dev, np.random.default_rng(d + page), dtype, interleaved, heads, kv_heads, d, dim, page, [1, 50, 40, 20, 40, 2, 33], [1, 50, 7, 0, 5, 4, 2], (4, 38 // page))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads, kv_heads, d, dim", [(2, 1, 64, 64), (1, 1, 20, 8), (4, 2, 40, 40), (1, 1, 7, 6)])
def test_many_into_the_cache(dev, dtype, interleaved, heads, kv_heads, d, dim):
    """several tokens to a block: of two sequences, of none, of pages that are missing"""
    lens, new = [700, 1, 900, 3, 333, 2, 64, 64], [600, 1, 700, 3, 111, 4, 1, 64]
    into_the_cache(dev, np.random.default_rng(d), dtype, interleaved, heads, kv_heads, d, dim, 16, lens, new, (2, 30))


@pytest.mark.parametrize("dtype", DTYPES)
def test_into_the_cache_is_the_two_calls(dev, dtype):
    """the same bits as rope_tokens of q and k and the append of what comes out"""
    rng = np.random.default_rng(5)
    heads, kv_heads, d = 8, 2, 64
    p = ref.Paged(rng, dtype, heads, kv_heads, d, 16, [900, 33, 1], [1, 33, 1])
    w = (heads + 2 * kv_heads) * d
    qkv = ref.upload(dev, rng.standard_normal((p.tokens, w)), dtype)
    q, k, v = (qkv.view(o * d, (p.tokens, n, d)) for o, n in ((0, heads), (heads, kv_heads), (heads + kv_heads, kv_heads)))
    a, b = (dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32))) for _ in range(2))
    starts, table, s = dev.upload(p.starts), dev.rope_table(d), dict(strides=(w, d))
    at = dev.upload(np.concatenate([p.lens[i] - p.new[i] + np.arange(p.new[i]) for i in range(3)]).astype(np.int32))
    out = dev.paged_rope_append(a, starts, q, k, v, table, q_strides=(w, d), k_strides=(w, d), v_strides=(w, d))
    want = dev.rope_tokens(q, at, table, **s)
    dev.paged_append(b, starts, dev.rope_tokens(k, at, table, **s), v, v_strides=(w, d))
    assert np.array_equal(out.to_numpy(), want.to_numpy())
    assert np.array_equal(a.k_pages.to_numpy(), b.k_pages.to_numpy()) and np.array_equal(a.v_pages.to_numpy(), b.v_pages.to_numpy())


def test_recorded(dev):
    rng = np.random.default_rng(6)
    x, positions = dev.upload(rng.standard_normal((5, 3, 64)).astype(np.float32)), dev.upload(np.arange(5, dtype=np.int32))
    table, out = dev.rope_table(64), dev.empty((5, 3, 64), _lib.F32)
    with dev.capture() as graph:
        dev.rope_tokens(x, positions, table, out=out)
    for base in (0, 77, 100000):
        positions.reshape((5,)).upload(np.arange(base, base + 5, dtype=np.int32))
        graph.launch()
        got = out.to_numpy()
        assert np.array_equal(dev.rope_tokens(x, positions, table).to_numpy(), got)
