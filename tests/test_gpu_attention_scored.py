"""Attention whose scores are capped, biased by distance, or masked by documents and prefixes, against its definition in 64 bits.

Bounds are attention_ref.py's with a score's error made larger by what is done to it (u = 2^-24): tanh has a slope of at most 1, and computed as 1 - 2 / (e^2y + 1) it is off by
2u |y| (1 - tanh^2) < u from the two products that make its argument, u from the exponential (off by 2u), 2u from the sum, 4u from the reciprocal (off by 2u) and u from the last
operation, in all 9u, with the cap's own rounding and that of log2(e) less than 12u of the cap.  In f32, and for a cap
above 1024 ln 2, a score below an eighth of the cap is a series or a polynomial of it, off by less than 16u of itself: 4u for what is left out, six roundings of a value and
four of constants.  A bias is off by the roundings of slope * log2(e), of the distance and of the sum, 4u of it and of the score."""
import numpy as np
import pytest

import attention_ref as ref
from attention_ref import U
from ratchet_amd import _lib

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def dev():
    from ratchet_amd import Device

    d = Device(0)
    yield d
    d.close()


def head(q, k, v, see, scale, dtype, cap=0.0, slope=0.0, distance=None):
    """o, lse and their bounds"""
    n, d = q.shape
    o, lse = np.zeros((n, v.shape[1])), np.full(n, -np.inf)
    o_off, lse_off = np.zeros_like(o), np.zeros(n)
    some = see.any(axis=1) if k.shape[0] else np.zeros(n, bool)
    if not some.any():
        return o, lse, o_off, lse_off
    k0, v0 = (np.where(see.any(axis=0)[:, None], x, 0.0) for x in (k, v))
    s = (q @ k0.T) * scale
    mass = np.where(see, np.abs(q) @ np.abs(k0).T, 0.0).max(axis=1) * abs(scale) * (d + 16) * U
    if cap:
        near = cap / 8 if dtype == "f32" or cap > 1024 / np.log2(np.e) else 0.0
        small = np.where(see & (np.abs(s) < near), np.minimum(12 * U * cap, 16 * U * np.abs(s)), np.where(see & (np.abs(s) < np.inf), 12 * U * cap, 0.0)).max(axis=1)
        s = cap * np.tanh(s / cap)
        mass = mass + small
    if slope:
        bias = slope * np.abs(distance)
        s = s - bias
        mass = mass + 4 * U * np.where(see, np.abs(bias) + np.abs(s), 0.0).max(axis=1)
    s = np.where(see, s, -np.inf)
    m = np.where(some, s.max(axis=1), 0.0)
    x = np.exp(s - m[:, None])
    total = np.where(some, x.sum(axis=1), 1.0)
    w = x / total[:, None]
    lse = np.where(some, np.log(total) + m, -np.inf)
    o, e, seen = w @ v0, ref.HALF_STEP[dtype], see.sum(axis=1)
    o_off = e * np.abs(o) + (e + 2 * mass + (2 * seen + 64) * U)[:, None] * (w @ np.abs(v0)) + ref.TINY[dtype]
    if dtype == "f16":
        o_off = o_off + 2.0 ** -25 * (see.astype(float) @ np.abs(v0))
    return o, lse, o_off, mass + (seen + 32) * U + 4 * U * np.abs(np.where(some, lse, 0.0))


def visible(n, keys, shift, causal, window, sinks, documents=None, prefix=None):
    """[n, keys] key by key: documents: the starts and the last end; prefix: a number, or one for each document"""
    see = np.zeros((n, keys), bool)
    for j in range(n):
        p = j + shift
        lo, hi, front = 0, keys, 0 if prefix is None or documents is not None else prefix
        if documents is not None:
            inside = [d for d in range(len(documents) - 1) if documents[d] <= p < documents[d + 1]]
            lo, hi = (documents[inside[0]], min(documents[inside[0] + 1], keys)) if inside else (0, 0)
            front = prefix[inside[0]] if inside and prefix is not None else 0
        t = np.arange(lo, max(lo, hi))
        back = t <= p
        if window:
            back &= (p - t < window) | (t - lo < sinks)
        see[j, t] = (back | (t - lo < front)) if causal else True
    return see


def dense(dev, rng, dtype, batch, heads, kv_heads, queries, keys, dim, causal=True, window=0, sinks=0, lens=None, cap=0.0, slopes=None, documents=None, prefix=None, spread=2.0,
          change=None, scale=None, aligned=True):
    q, k, v = (ref.rounded(rng.standard_normal(s) * x, dtype) for s, x in (((batch, heads, queries, dim), spread), ((batch, kv_heads, keys, dim), 1.0), ((batch, kv_heads, keys, dim), 1.0)))
    if change:
        change(q, k, v)
    scale = dim ** -0.5 if scale is None else scale
    ints = lambda x: None if x is None else dev.upload(np.asarray(x, np.int32))        # noqa: E731
    lse = dev.empty((batch, heads, queries), _lib.F32)
    on = []
    for x in (q, k, v):
        if aligned:
            on.append(ref.upload(dev, x, dtype))
        else:                                                   # an element off the vector grid: the kernel for any layout
            on.append(ref.upload(dev, np.concatenate([[0.0], x.ravel()]), dtype).view(1, x.shape))
    out = dev.attention(*on, lens=ints(lens), causal=causal, window=window, sinks=sinks, scale=scale, lse=lse, cap=cap, slopes=None if slopes is None else dev.upload(np.asarray(slopes, np.float32)),
                        documents=ints(documents), prefix=ints(prefix))
    got, got_lse = ref.values(out.to_numpy(), dtype), lse.to_numpy()
    for b in range(batch):
        n = keys if lens is None else int(np.clip(lens[b], 0, keys))
        shift = n - queries
        see = visible(queries, n, shift, causal, window, sinks, None if documents is None else documents[b], None if prefix is None else prefix[b])
        distance = (np.arange(queries) + shift)[:, None] - np.arange(n)[None, :]
        for h in range(heads):
            g = h // (heads // kv_heads)
            o, want_lse, o_off, lse_off = head(q[b, h], k[b, g, :n], v[b, g, :n], see, scale, dtype, cap, 0.0 if slopes is None else float(np.float32(slopes[h])), distance)
            ref.check(got[b, h], o, o_off, ("o", b, h))
            ref.check(got_lse[b, h], want_lse, lse_off, ("lse", b, h))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("queries, keys", [(1, 150), (1, 3000), (100, 150)])
def test_visible_values_that_are_not_finite(dev, dtype, bad, queries, keys):
    """a value that is seen makes its columns what it is, and others stay right"""
    q, k, v = (ref.rounded(np.random.default_rng(1).standard_normal(s), dtype) for s in ((2, 4, queries, 64), (2, 2, keys, 64), (2, 2, keys, 64)))
    v[0, 1, 70, 5] = bad
    out = ref.values(dev.attention(*(ref.upload(dev, x, dtype) for x in (q, k, v)), cap=5.0, causal=False).to_numpy(), dtype)
    clean = ref.values(dev.attention(*(ref.upload(dev, x, dtype) for x in (q, k, np.where(np.isfinite(v), v, 0.0))), cap=5.0, causal=False).to_numpy(), dtype)
    got = out[0, 2:, :, 5]
    assert np.isnan(got).all() if bad != bad else (got == bad).all()
    clean[0, 2:, :, 5] = out[0, 2:, :, 5] = 0.0
    assert np.isfinite(out).all()
    # both are within the bound of the definition's result, whose weights sum to 1
    mass = (np.abs(q) @ np.abs(k).repeat(2, 1).transpose(0, 1, 3, 2)).max() / 8 * 80 * U + 60 * U
    off = (2 * ref.HALF_STEP[dtype] + 2 * mass + (2 * keys + 64) * U + (keys * 2.0 ** -25 if dtype == "f16" else 0.0)) * np.abs(v[np.isfinite(v)]).max() + ref.TINY[dtype]
    assert (np.abs(out - clean) <= 2 * off).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, queries", [(16, 1, 1), (17, 1, 1), (12, 4, 1), (5, 1, 3), (8, 8, 1), (8, 8, 16), (4, 2, 8), (4, 2, 9), (3, 3, 2)])
@pytest.mark.parametrize("dim", [64, 96, 40])
def test_a_few_rows(dev, dtype, heads, kv_heads, queries, dim):
    rng = np.random.default_rng(heads + queries)
    for keys in (1, 63, 64, 65, 700, 2100):
        dense(dev, rng, dtype, 2, heads, kv_heads, queries, keys, dim, cap=15.0, slopes=alibi(heads), window=0 if keys < 700 else 500, sinks=3)


def alibi(heads):
    return 2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cap, biased", [(5.0, False), (50.0, False), (0.0, True), (20.0, True), (1e-3, False), (300.0, False), (1e4, True), (1e30, False)])
@pytest.mark.parametrize("queries, keys, causal", [(1, 1, True), (1, 777, True), (3, 65, False), (130, 300, True), (64, 64, True), (5, 3, True), (200, 90, False)])
def test_cap_and_bias(dev, dtype, cap, biased, queries, keys, causal):
    dense(dev, np.random.default_rng(keys), dtype, 2, 4, 2, queries, keys, 64, causal=causal, cap=cap, slopes=alibi(4) if biased else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 20, 40, 64, 80, 96, 112, 128, 192, 256, 264])
@pytest.mark.parametrize("queries", [1, 67])
def test_head_dims(dev, dtype, dim, queries):
    rng = np.random.default_rng(dim)
    dense(dev, rng, dtype, 2, 4, 2, queries, 131, dim, cap=7.0, slopes=alibi(4), window=50, sinks=3)
    dense(dev, rng, dtype, 1, 2, 2, queries, 131, dim, documents=[[0, 30, 100, 120]], prefix=[[9, 40, 20]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("queries, keys, documents", [
    (300, 300, [[0, 300], [0, 120]]), (300, 300, [[0, 1, 2, 3, 64, 64, 64, 200, 300], [5, 70, 70, 71, 140, 150, 150, 151, 290]]), (300, 300, [[300, 300], [0, 0]]),
    (1, 500, [[0, 100, 400, 500], [0, 10, 499, 500]]), (1, 500, [[0, 100, 400, 499], [3, 3, 3, 3]]), (140, 500, [[0, 365, 430, 470], [400, 401, 402, 450]]),
    (40, 20, [[0, 7, 20], [0, 20, 25]]), (129, 129, [list(range(130)), [0] * 65 + list(range(64, 129))])])
def test_documents(dev, dtype, causal, queries, keys, documents):
    rng = np.random.default_rng(queries + keys)
    dense(dev, rng, dtype, 2, 4, 2, queries, keys, 64, causal=causal, documents=documents)
    dense(dev, rng, dtype, 2, 4, 4, queries, keys, 20, causal=causal, documents=documents, cap=9.0, aligned=False)
    if causal:
        dense(dev, rng, dtype, 2, 4, 1, queries, keys, 128, documents=documents, window=33, sinks=5, slopes=alibi(4))
        prefix = rng.integers(0, 90, (2, len(documents[0]) - 1))
        dense(dev, rng, dtype, 2, 2, 2, queries, keys, 32, documents=documents, prefix=prefix)
        dense(dev, rng, dtype, 2, 2, 2, queries, keys, 32, documents=documents, prefix=prefix, window=20, sinks=2)
        dense(dev, rng, dtype, 2, 2, 2, queries, keys, 32, documents=documents, prefix=prefix, window=20, sinks=2, aligned=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries, keys", [(1, 700), (200, 200), (150, 333), (30, 10)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (40, 0), (64, 70)])
def test_prefix(dev, dtype, queries, keys, window, sinks):
    rng = np.random.default_rng(queries)
    dense(dev, rng, dtype, 4, 4, 2, queries, keys, 80, window=window, sinks=sinks, prefix=[0, 1, 150, 100000])
    dense(dev, rng, dtype, 4, 4, 2, queries, keys, 80, window=window, sinks=sinks, prefix=[-5, 64, 65, 7], aligned=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_lens_of_a_padded_batch(dev, dtype, causal):
    rng = np.random.default_rng(7)
    lens = [0, 1, 5, 149, 150, 1000, -3]
    for queries in (1, 9, 140):
        dense(dev, rng, dtype, 7, 4, 2, queries, 150, 48, causal=causal, lens=lens, cap=30.0, slopes=alibi(4))
        dense(dev, rng, dtype, 7, 4, 2, queries, 150, 48, causal=causal, lens=lens, documents=[[0, 3, 140, 150]] * 7, prefix=[[2, 100, 5]] * 7 if causal else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_hidden_keys_hold_anything(dev, dtype, bad, aligned):
    def change(q, k, v):
        k[:, :, 100:130], v[:, :, 100:130] = bad, bad

    rng = np.random.default_rng(3)
    # the keys of the middle document, which no query of the last one sees; and keys beyond a window behind a prefix
    dense(dev, rng, dtype, 1, 2, 2, 60, 200, 64, documents=[[0, 100, 130, 200]], change=change, cap=5.0, aligned=aligned)
    dense(dev, rng, dtype, 1, 2, 2, 40, 200, 64, window=20, prefix=[80], change=change, slopes=alibi(2), aligned=aligned)
    # the same for a few rows
    dense(dev, rng, dtype, 2, 4, 2, 1, 200, 64, documents=[[0, 100, 130, 200], [0, 130, 199, 200]], change=change, cap=5.0, aligned=aligned)
    dense(dev, rng, dtype, 2, 6, 2, 3, 200, 64, window=20, prefix=[80, 3], change=change, slopes=alibi(6), aligned=aligned)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cap", [1e3, 3e4, 1e6, 1e12, 1e18])
def test_a_large_cap_that_one_row_reaches(dev, dtype, cap):
    """next to rows whose scores are ordinary: every 16th query's first column is about the cap, as far as the type holds it"""
    def change(q, k, v):
        most = min(cap, 3e4) if dtype == "f16" else cap
        q[0, 0, 3::16, 0] = np.float32(2.0 ** np.floor(np.log2(most)))
        k[0, 0, 5::7, 0] = 4.0
        k[0, 0, 6::7, 0] = -4.0
    dense(dev, np.random.default_rng(5), dtype, 1, 2, 1, 90, 130, 64, cap=cap, change=change)
    dense(dev, np.random.default_rng(5), dtype, 1, 2, 1, 5, 130, 64, cap=cap, change=change)
    dense(dev, np.random.default_rng(5), dtype, 1, 2, 1, 40, 70, 20, cap=cap, change=change, aligned=False)
    if cap in (1e3, 1e6):                                       # keys shared out, rows of other tiles behind the ones that are computed again; 17 heads of a KV head
        dense(dev, np.random.default_rng(6), dtype, 1, 2, 1, 200, 3000, 64, cap=cap, change=change)
        dense(dev, np.random.default_rng(7), dtype, 1, 17, 1, 17, 2000, 80, cap=cap, change=change, slopes=alibi(17), causal=False)
        dense(dev, np.random.default_rng(8), dtype, 1, 17, 1, 1, 2000, 128, cap=cap, change=lambda q, k, v: change(np.swapaxes(q, 1, 2), k, v))


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_are_infinite_are_capped(dev, dtype):
    """a column of +-1 where it is not large: of odd queries and every third key, whose products pass f32's largest (f16: 3.6e9) or reach the cap anyhow"""
    rng = np.random.default_rng(5)
    q, k, v = (ref.rounded(rng.standard_normal(s), dtype) for s in ((1, 2, 30, 64), (1, 2, 70, 64), (1, 2, 70, 64)))
    large = 6e4 if dtype == "f16" else 3e38
    q[..., 0], k[..., 0] = np.sign(q[..., 0]), np.sign(k[..., 0])
    q[:, :, 1::2, 0] *= large
    k[:, :, ::3, 0] *= large
    q, k = ref.rounded(q, dtype), ref.rounded(k, dtype)
    out = dev.attention(ref.upload(dev, q, dtype), ref.upload(dev, k, dtype), ref.upload(dev, v, dtype), cap=4.0, causal=False)
    s = np.matmul(q, k.transpose(0, 1, 3, 2)) / 8
    w = np.exp(4.0 * np.tanh(s / 4.0))
    want = np.matmul(w / w.sum(axis=-1, keepdims=True), v)
    # scores are off by their products' sums where they are small, and by nothing but the cap's roundings where they are large
    mass = np.where(np.abs(s) < 100, np.abs(q) @ np.abs(k).transpose(0, 1, 3, 2), 0.0).max() / 8 * 80 * U + 48 * U
    off = (ref.HALF_STEP[dtype] * 2 + 2 * mass + 204 * U) * np.abs(v).max() + 70 * 2.0 ** -25
    ref.check(ref.values(out.to_numpy(), dtype), want, off, "capped")


def test_negative_scale(dev):
    for dtype in DTYPES:
        dense(dev, np.random.default_rng(9), dtype, 1, 2, 1, 70, 100, 64, scale=-0.2, cap=3.0, slopes=alibi(2))
        dense(dev, np.random.default_rng(9), dtype, 1, 2, 1, 70, 100, 64, scale=-0.2, prefix=[40], aligned=False, cap=3.0)


def test_long_walks_are_shared_out_and_joined(dev):
    rng = np.random.default_rng(11)
    for dtype in DTYPES:
        dense(dev, rng, dtype, 1, 2, 1, 1, 5000, 64, cap=20.0, slopes=[1e-3, 1e-4])
        dense(dev, rng, dtype, 1, 2, 1, 200, 3000, 64, cap=20.0, prefix=[2950])
        dense(dev, rng, dtype, 1, 2, 1, 1, 5000, 64, documents=[[0, 17, 4000, 5000]], window=700, sinks=80)
        dense(dev, rng, dtype, 2, 1, 1, 300, 3000, 64, documents=[[0, 1003, 2800, 3000], [0, 2705, 2900, 2950]], prefix=[[700, 900, 100], [2700, 3, 0]], window=64, sinks=4)


def paged(dev, rng, dtype, heads, kv_heads, dim, page, lens, new, window=0, sinks=0, cap=0.0, slopes=None, prefix=None, holes=(), aligned=True):
    p = ref.Paged(rng, dtype, heads, kv_heads, dim, page, lens, new, spread=2.0, holes=holes)
    scale = dim ** -0.5
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    lse = dev.empty((p.tokens, heads), _lib.F32)
    q = ref.upload(dev, p.q, dtype) if aligned else ref.upload(dev, np.concatenate([[0.0], p.q.ravel()]), dtype).view(1, p.q.shape)
    out = dev.paged_attention(q, cache, dev.upload(p.starts), window=window, sinks=sinks, lse=lse, cap=cap, slopes=None if slopes is None else dev.upload(np.asarray(slopes, np.float32)),
                              prefix=None if prefix is None else dev.upload(np.asarray(prefix, np.int32)))
    got, got_lse = ref.values(out.to_numpy(), dtype), lse.to_numpy()
    for b in range(len(p.lens)):
        lo, hi = p.starts[b], p.starts[b + 1]
        k, gone = p.rows(p.k, b)
        v, _ = p.rows(p.v, b)
        keys, shift = k.shape[1], int(max(p.lens[b], 0)) - int(hi - lo)
        see = visible(hi - lo, keys, shift, True, window, sinks, None, None if prefix is None else prefix[b]) & ~gone[None, :]
        distance = (np.arange(hi - lo) + shift)[:, None] - np.arange(keys)[None, :]
        for h in range(heads):
            g = h // (heads // kv_heads)
            o, want_lse, o_off, lse_off = head(p.q[lo:hi, h], k[g], v[g], see, scale, dtype, cap, 0.0 if slopes is None else float(np.float32(slopes[h])), distance)
            ref.check(got[lo:hi, h], o, o_off, ("o", b, h))
            ref.check(got_lse[lo:hi, h], want_lse, lse_off, ("lse", b, h))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("options", [dict(cap=20.0), dict(slopes=alibi(8)), dict(cap=50.0, slopes=alibi(8), window=100, sinks=3), dict(prefix=[0, 5, 300, 64, 10 ** 6, -1]),
                                     dict(prefix=[700, 1, 0, 17, 40, 2], window=33, sinks=20), dict(cap=9.0, prefix=[64] * 6, window=64)])
def test_paged(dev, dtype, options, aligned):
    rng = np.random.default_rng(1)
    paged(dev, rng, dtype, 8, 2, 64, 16, [1, 700, 33, 64, 250, 2], [1, 1, 1, 1, 1, 1], holes=[(1, 3)], aligned=aligned, **options)
    paged(dev, rng, dtype, 8, 2, 64, 24, [1, 700, 33, 64, 250, 2], [1, 150, 0, 64, 1, 4], holes=[(1, 3)], aligned=aligned, **options)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 80, 96, 128, 192, 256])
def test_paged_head_dims(dev, dtype, dim):
    rng = np.random.default_rng(dim)
    paged(dev, rng, dtype, 4, 1, dim, 16, [300, 1, 90], [1, 1, 1], cap=10.0, slopes=alibi(4), prefix=[3, 0, 100])
    paged(dev, rng, dtype, 4, 1, dim, 16, [300, 1, 90], [90, 1, 90], cap=10.0, slopes=alibi(4), prefix=[3, 0, 100])


def test_nothing_changed_is_the_plain_call(dev):
    """no cap, slopes, documents or prefix: the plain call's bits"""
    import ctypes

    rng = np.random.default_rng(2)
    q, k, v = (dev.upload(rng.standard_normal(s).astype(np.float16)) for s in ((2, 4, 70, 64), (2, 2, 90, 64), (2, 2, 90, 64)))
    want = dev.attention(q, k, v).to_numpy()
    out = dev.empty(q.shape, _lib.F16)
    u4 = lambda s: (ctypes.c_uint32 * 4)(*s)        # noqa: E731
    assert dev.lib.rt_attention_scored(dev.handle, _lib.F16, q.ptr, u4(q.shape), None, k.ptr, None, v.ptr, None, u4(k.shape), None, out.ptr, None, None, 0.125, 1, 0, 0,
                                       ctypes.byref(_lib.Scores())) == 0
    assert np.array_equal(out.to_numpy().view(np.uint16), want.view(np.uint16))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_recorded_calls(dev, dtype):
    """a replay reads documents, prefixes and slopes as they then are; calls that share the workspace"""
    rng = np.random.default_rng(4)
    q, k, v = (ref.upload(dev, rng.standard_normal(s), dtype) for s in ((1, 4, 1, 64), (1, 2, 3000, 64), (1, 2, 3000, 64)))
    documents, prefix, slopes = dev.upload(np.array([[0, 1000, 3000]], np.int32)), dev.upload(np.array([10], np.int32)), dev.upload(alibi(4).astype(np.float32))
    one, two = dev.empty(q.shape, q.dt), dev.empty(q.shape, q.dt)

    def calls():
        dev.attention(q, k, v, documents=documents, out=one)
        dev.attention(q, k, v, cap=5.0, slopes=slopes, prefix=prefix, window=100, out=two)

    calls()
    with dev.capture() as graph:
        calls()
    for start in (0, 2999, 1500, 700):
        documents.reshape((1, 3)).upload(np.array([[0, start, 3000]], np.int32))
        prefix.reshape((1,)).upload(np.array([start], np.int32))
        calls()
        want = one.to_numpy(), two.to_numpy()
        one.zero_()
        two.zero_()
        graph.launch()
        assert np.array_equal(one.to_numpy(), want[0]) and np.array_equal(two.to_numpy(), want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extra", [0, 40])
def test_rows_of_no_sequence_stay_as_they_were(dev, dtype, extra):
    """rows in front of the first sequence's and behind the last one's; with none extra the call is one of few rows"""
    rng = np.random.default_rng(6)
    p = ref.Paged(rng, dtype, 4, 2, 64, 16, [900, 40, 7, 300, 1, 64], [1, 0, 1, 1, 0, 0])
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    tokens = 6 + extra
    q = np.full((tokens, 4, 64), np.nan)
    q[2:5] = p.q
    out, lse = ref.upload(dev, np.full(q.shape, 3.0), dtype), dev.upload(np.full((tokens, 4), 3.0, np.float32))
    dev.paged_attention(ref.upload(dev, q, dtype), cache, dev.upload(p.starts + 2), out=out, lse=lse, cap=9.0)
    got, got_lse = ref.values(out.to_numpy(), dtype), lse.to_numpy()
    assert (got[:2] == 3).all() and (got[5:] == 3).all() and (got_lse[:2] == 3).all() and (got_lse[5:] == 3).all()
    for row, b in ((2, 0), (3, 2), (4, 3)):
        k, _ = p.rows(p.k, b)
        v, _ = p.rows(p.v, b)
        for h in range(4):
            o, want_lse, o_off, lse_off = head(q[row:row + 1, h], k[h // 2], v[h // 2], np.ones((1, k.shape[1]), bool), 0.125, dtype, 9.0)
            ref.check(got[row:row + 1, h], o, o_off, ("o", b, h))
            ref.check(got_lse[row:row + 1, h], want_lse, lse_off, ("lse", b, h))


def test_starts_and_texts_that_decrease_leave_later_calls_right(dev):
    """what they give is nobody's, but the counters of a launch are 0 again"""
    rng = np.random.default_rng(7)
    p = ref.Paged(rng, "f16", 4, 2, 64, 16, [3000, 2500, 2000, 1500], [1, 1, 1, 1])
    cache = dev.paged_cache(ref.upload(dev, p.k, "f16"), ref.upload(dev, p.v, "f16"), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    q, right = ref.upload(dev, p.q, "f16"), dev.upload(p.starts)
    want = dev.paged_attention(q, cache, right, cap=5.0).to_numpy()
    k = ref.upload(dev, rng.standard_normal((1, 2, 3000, 64)), "f16")
    one, many = (ref.upload(dev, rng.standard_normal((1, 4, n, 64)), "f16") for n in (1, 200))
    sane = dev.upload(np.array([[0, 1000, 2990, 3000]], np.int32))
    whole = [dev.attention(x, k, k, documents=sane, window=300, sinks=9).to_numpy() for x in (one, many)]
    for bad in ([4, 0, 3, 1, 2], [0, 4, 0, 4, 0], [3, 1, 2, 0, 4], [-5, 100, -7, 9, 2]):
        dev.paged_attention(q, cache, dev.upload(np.array(bad, np.int32)), cap=5.0)
        assert np.array_equal(dev.paged_attention(q, cache, right, cap=5.0).to_numpy(), want)
    for bad in ([3000, 0, 2000, 100], [50, 10, 3000, -4], [-100, 5000, 200, 9999], [0, 0, 0, 0]):
        texts = dev.upload(np.array([bad], np.int32))
        for x, w in zip((one, many), whole):
            for window in (0, 300):
                dev.attention(x, k, k, documents=texts, window=window, sinks=9 if window else 0)
            assert np.array_equal(dev.attention(x, k, k, documents=sane, window=300, sinks=9).to_numpy(), w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_texts(dev, dtype):
    """more than the lanes of a wave, and texts of one token"""
    rng = np.random.default_rng(8)
    for n in (62, 63, 64, 65, 200):
        cuts = np.sort(rng.integers(0, 401, n - 1))
        documents = [np.concatenate([[0], cuts, [400]]).tolist(), np.concatenate([[3], np.sort(rng.integers(3, 350, n - 1)), [350]]).tolist()]
        prefix = rng.integers(0, 8, (2, n))
        dense(dev, rng, dtype, 2, 2, 1, 400, 400, 64, documents=documents, prefix=prefix)
        dense(dev, rng, dtype, 2, 2, 1, 1, 400, 64, documents=documents, prefix=prefix, cap=4.0)
        dense(dev, rng, dtype, 2, 2, 1, 90, 400, 64, documents=documents, aligned=False, slopes=alibi(2))


@pytest.mark.parametrize("dtype", DTYPES)
def test_scale_of_zero_and_next_to_it(dev, dtype):
    """the bias alone decides"""
    for scale in (0.0, 1e-20, -1e-13, 1e-11):
        for queries in (1, 70):
            dense(dev, np.random.default_rng(9), dtype, 1, 4, 2, queries, 130, 64, scale=scale, slopes=alibi(4))
            dense(dev, np.random.default_rng(9), dtype, 1, 4, 2, queries, 130, 64, scale=scale, cap=2.0)
