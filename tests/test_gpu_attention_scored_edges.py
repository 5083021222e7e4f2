"""Attention with changed scores where its numbers end."""
import numpy as np
import pytest

import attention_ref as ref
from attention_ref import U
from ratchet_amd import _lib
from test_gpu_attention_scored import dense, head, paged

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def dev():
    from ratchet_amd import Device

    d = Device(0)
    yield d
    d.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("queries", [1, 70])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("cap", [1.0e38, 1.17e38])
def test_the_largest_caps(dev, dtype, queries, aligned, cap):
    """scores of 1.7 cap and its half, its 64th and its negative among those that are 0: the largest has all the weight, and its row is the result.  Products are powers of two,
    so lse is off by the cap's 12 u (test_gpu_attention_scored.py), 2 u of 1.7 cap for the division by the cap, and 4 u for units and the last product: 24 u of the cap"""
    rng, d, keys = np.random.default_rng(1), 64, 130
    q, k, v = np.zeros((1, 2, queries, d)), np.zeros((1, 1, keys, d)), ref.rounded(rng.standard_normal((1, 1, keys, d)), dtype)
    q[..., 0] = 2.0 ** 60
    q[0, 1, :, 0] = -2.0 ** 60                                   # the other head's signs are turned
    top = 2.0 ** 67 / 8
    k[0, 0, [7, 70, 100, 129], 0] = top, top / 2, top / 64, -top
    parts = []
    for x in (q, k, v):
        parts.append(ref.upload(dev, x, dtype) if aligned else ref.upload(dev, np.concatenate([[0.0], x.ravel()]), dtype).view(1, x.shape))
    lse = dev.empty((1, 2, queries), _lib.F32)
    out = ref.values(dev.attention(*parts, causal=False, scale=8.0, cap=cap, lse=lse).to_numpy(), dtype)
    most = float(np.float32(cap)) * np.tanh(8.0 * 2.0 ** 60 * top / float(np.float32(cap)))
    assert np.array_equal(out[0, 0], np.broadcast_to(v[0, 0, 7], (queries, d))) and np.array_equal(out[0, 1], np.broadcast_to(v[0, 0, 129], (queries, d)))
    assert (np.abs(lse.to_numpy() - most) <= 24 * U * cap).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 70])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("slope, scale", [(3e37, 0.125), (2.3e38, 0.125), (2.5e38, -0.125), (3.4028234e38, 0.125), (1e34, 1e-5)])
def test_a_slope_that_leaves_a_row_its_own_key(dev, dtype, queries, aligned, cap, slope, scale):
    """next to a head of the same KV head whose slope is ordinary; the bounds are test_gpu_attention_scored.py's, the first head's for a row of one visible key"""
    rng, keys, d = np.random.default_rng(2), 130, 64
    q, k, v = (ref.rounded(rng.standard_normal(s), dtype) for s in ((1, 2, queries, d), (1, 1, keys, d), (1, 1, keys, d)))
    parts = []
    for x in (q, k, v):
        parts.append(ref.upload(dev, x, dtype) if aligned else ref.upload(dev, np.concatenate([[0.0], x.ravel()]), dtype).view(1, x.shape))
    slopes, lse = np.array([slope, 0.125], np.float32), dev.empty((1, 2, queries), _lib.F32)
    out = ref.values(dev.attention(*parts, scale=scale, cap=cap, slopes=dev.upload(slopes), lse=lse).to_numpy(), dtype)
    distance = (np.arange(queries) + keys - queries)[:, None] - np.arange(keys)[None, :]
    for h, (see, s) in enumerate(((distance == 0, 0.0), (distance >= 0, 0.125))):
        o, want_lse, o_off, lse_off = head(q[0, h], k[0, 0], v[0, 0], see, scale, dtype, cap, s, distance)
        ref.check(out[0, h], o, o_off, ("o", h))
        ref.check(lse.to_numpy()[0, h], want_lse, lse_off, ("lse", h))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [63, 64, 3000])
def test_texts_padded_with_ends(dev, dtype, n):
    """an array of a fixed length whose last texts hold nothing, queries behind them all, and texts of nothing in front and between"""
    rng = np.random.default_rng(n)
    few = [0, 0, 0, 40, 41, 41, 41, 41, 130, 350]
    some = [5] * 30 + np.sort(rng.integers(5, 300, 20)).tolist()
    documents = [few + [350] * (n + 1 - len(few)), some + [some[-1]] * (n + 1 - len(some))]
    prefix = rng.integers(0, 30, (2, n))
    dense(dev, rng, dtype, 2, 2, 1, 400, 400, 64, documents=documents, prefix=prefix)
    dense(dev, rng, dtype, 2, 4, 2, 100, 340, 64, documents=documents, window=17, sinks=2, cap=5.0)
    dense(dev, rng, dtype, 2, 2, 1, 8, 304, 64, documents=documents, prefix=prefix)
    dense(dev, rng, dtype, 2, 2, 1, 8, 352, 64, documents=documents, causal=False)
    dense(dev, rng, dtype, 2, 2, 1, 30, 360, 64, documents=documents, aligned=False)


def large_keys_that_some_rows_do_not_see(q, k, v):
    """the first text's keys are large and its queries 0, so that its scores are 0 and those of the second text's rows, which do not see them, are far beyond a cap"""
    q[:, :, :70] = 0.0
    k[:, :, :70] *= 2.0 ** 12


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("cap", [1e3, 1e7])
def test_large_keys_that_no_other_row_sees(dev, dtype, dim, cap):
    rng = np.random.default_rng(dim)
    dense(dev, rng, dtype, 1, 2, 1, 200, 200, dim, documents=[[0, 70, 200]], cap=cap, change=large_keys_that_some_rows_do_not_see)
    dense(dev, rng, dtype, 1, 2, 1, 200, 200, dim, documents=[[0, 70, 190]], prefix=[[9, 90]], window=40, sinks=3, slopes=[0.5, 0.01], cap=cap, change=large_keys_that_some_rows_do_not_see)
    # keys behind the window of all rows but the first, whose query is 0
    def first(q, k, v):
        q[:, :, 0] = 0.0
        k[:, :, 1] *= 2.0 ** 12
    dense(dev, rng, dtype, 1, 2, 1, 40, 70, dim, window=30, cap=cap, change=first)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("what", ["hidden keys", "no scale"])
def test_rows_are_computed_again_for_what_they_see_alone(dev, dtype, what):
    """Computed again a row at a time, this call takes 125 times as long (20 us, 2.5 ms): scores beyond a large cap that no row sees, or that a scale of 0 makes 0, have no part in that"""
    def took(hidden, scale):
        rng = np.random.default_rng(3)
        q, k, v = (rng.standard_normal((1, 8, 1024, 64)) for _ in range(3))
        if hidden:
            large_keys_that_some_rows_do_not_see(q, k, v)
        parts, documents, out = [ref.upload(dev, x, dtype) for x in (q, k, v)], dev.upload(np.array([[0, 70, 1024]], np.int32)), None
        times = []
        for _ in range(8):
            start, stop = dev.event(), dev.event()
            start.record()
            for _ in range(5):
                out = dev.attention(*parts, documents=documents, cap=1e4, scale=scale, out=out)
            stop.record()
            times.append(start.elapsed_ms(stop))
        return min(times)

    usual = took(False, 0.125)
    assert took(*((True, 0.125) if what == "hidden keys" else (False, 0.0))) < 3 * usual


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, dim", [(8, 2, 64), (16, 1, 64), (3, 1, 128), (6, 2, 40)])
def test_one_sequence_has_most_of_the_tokens(dev, dtype, heads, kv_heads, dim):
    """no more tokens than sequences, whose average is one, and several row tiles of one of them: whole and partial ones, whole walks and shared ones"""
    rng = np.random.default_rng(heads + dim)
    new = [0, 33, 0, 1, 2, 0, 1] + [0] * 33
    slopes = 2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)
    long, short = [5, 2500, 0, 700, 65, 0, 1] + [0] * 33, [0, 40, 0, 3, 64, 9, 1] + [0] * 33
    paged(dev, rng, dtype, heads, kv_heads, dim, 16, long, new, cap=20.0, slopes=slopes)
    paged(dev, rng, dtype, heads, kv_heads, dim, 24, long, new, window=100, sinks=3, slopes=slopes, holes=[(1, 3), (3, 0)])
    paged(dev, rng, dtype, heads, kv_heads, dim, 16, long, new, prefix=[0, 2490, 0, 5, 64] + [0] * 35, window=64, cap=9.0)
    paged(dev, rng, dtype, heads, kv_heads, dim, 16, short, new, cap=20.0, prefix=[3, 39, 1, 0, 64] + [7] * 35)
    paged(dev, rng, dtype, heads, kv_heads, dim, 16, [30] + short[1:], [40] + [0] * 39, slopes=slopes)           # more tokens than the sequence has


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("queries", [1, 70])
def test_a_bias_at_a_negative_scale(dev, dtype, aligned, queries):
    rng = np.random.default_rng(queries)
    for scale in (-0.2, -1e-6):
        dense(dev, rng, dtype, 2, 4, 2, queries, 200, 64, scale=scale, slopes=[0.5, 0.1, 0.02, 0.0], aligned=aligned)
        dense(dev, rng, dtype, 2, 4, 2, queries, 200, 96, scale=scale, slopes=[0.5, 0.1, -0.02, 1.0], window=30, sinks=2, aligned=aligned)
        dense(dev, rng, dtype, 1, 2, 2, queries, 200, 64, scale=scale, slopes=[0.5, 0.1], causal=False, aligned=aligned)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [1, 90, 0]])
def test_pages_at_a_negative_scale(dev, dtype, new):
    """the bits of the opposite queries at the positive one"""
    rng = np.random.default_rng(4)
    p = ref.Paged(rng, dtype, 8, 2, 64, 16, [700, 150, 33], new)
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    starts, slopes = dev.upload(p.starts), dev.upload((2.0 ** -np.arange(1, 9)).astype(np.float32))
    for options in (dict(), dict(cap=5.0), dict(window=40, sinks=3)):
        one, two = (dev.paged_attention(ref.upload(dev, q, dtype), cache, starts, scale=scale, slopes=slopes, **options).to_numpy() for q, scale in ((p.q, -0.2), (-p.q, 0.2)))
        assert np.array_equal(one.view(np.uint8), two.view(np.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [4, 8, 12, 16, 24, 32, 48, 56, 72, 88, 104, 120, 136, 144, 200])
def test_few_rows_of_any_columns(dev, dtype, dim):
    """head dims without a variant of their own, whose last products differ: contiguous and paged, walks of one and of several tiles and pieces"""
    rng = np.random.default_rng(dim)
    for keys in (1, 64, 65, 130, 700, 1500):
        dense(dev, rng, dtype, 2, 4, 2, 1, keys, dim, cap=15.0)
        dense(dev, rng, dtype, 1, 3, 1, 5, keys, dim, slopes=[0.5, 0.1, 0.01], causal=False)
    dense(dev, rng, dtype, 1, 2, 1, 8, 300, dim, documents=[[0, 100, 293, 300]], prefix=[[3, 50, 1]])
    paged(dev, rng, dtype, 4, 2, dim, 16, [700, 64, 65, 1], [1, 1, 1, 1], cap=15.0)
