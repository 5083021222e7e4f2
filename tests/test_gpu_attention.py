"""Attention over contiguous and paged keys against its definition in 64 bits: types, head dims and layouts, lengths from none to long ones,
windows and sinks, rows that see nothing, values in hidden places, strides.  The bounds are derived in attention_ref.py."""
import numpy as np
import pytest

import attention_ref as ref
from ratchet_amd import _lib

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def dev():
    from ratchet_amd import Device

    d = Device(0)
    yield d
    d.close()


def dense(dev, rng, dtype, batch, heads, kv_heads, queries, keys, dim, causal=True, window=0, sinks=0, lens=None, scale=None, change=None, spread=1.0):
    q, k, v = (ref.rounded(rng.standard_normal(s) * x, dtype) for s, x in (((batch, heads, queries, dim), spread), ((batch, kv_heads, keys, dim), 1.0), ((batch, kv_heads, keys, dim), 1.0)))
    if change:
        change(q, k, v)
    scale = dim ** -0.5 if scale is None else scale
    lse = dev.empty((batch, heads, queries), _lib.F32)
    out = dev.attention(ref.upload(dev, q, dtype), ref.upload(dev, k, dtype), ref.upload(dev, v, dtype), lens=None if lens is None else dev.upload(np.asarray(lens, np.int32)),
                        causal=causal, window=window, sinks=sinks, scale=scale, lse=lse)
    got, got_lse = ref.values(out.to_numpy(), dtype), lse.to_numpy()
    for b in range(batch):
        n = keys if lens is None else int(np.clip(lens[b], 0, keys))
        see = ref.visible(queries, n, n - queries, causal, window, sinks)
        for h in range(heads):
            g = h // (heads // kv_heads)
            o, want_lse, _, o_off, lse_off, _ = ref.head(q[b, h], k[b, g, :n], v[b, g, :n], see, scale, dtype)
            ref.check(got[b, h], o, o_off, ("o", b, h))
            ref.check(got_lse[b, h], want_lse, lse_off, ("lse", b, h))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 8, 20, 40, 64, 80, 96, 128, 192, 256, 264, 512])
def test_head_dims(dev, dtype, dim):
    dense(dev, np.random.default_rng(dim), dtype, 2, 4, 2, 67, 67, dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries, keys", [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (1, 1000), (2, 2), (3, 130), (16, 16), (17, 33), (32, 257), (33, 31), (64, 64), (65, 1),
                                           (127, 128), (128, 128), (129, 129), (200, 333), (300, 300)])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(dev, dtype, queries, keys, causal):
    dense(dev, np.random.default_rng(queries * 1000 + keys), dtype, 1, 2, 1, queries, keys, 64, causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (6, 6), (8, 2), (32, 2), (12, 4), (5, 1), (40, 1), (7, 7)])
def test_head_layouts(dev, dtype, heads, kv_heads):
    rng = np.random.default_rng(heads)
    dense(dev, rng, dtype, 2, heads, kv_heads, 19, 83, 40)
    dense(dev, rng, dtype, 2, heads, kv_heads, 1, 83, 40)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (64, 64), (65, 4), (100, 130), (1000, 4), (2 ** 32 - 1, 2 ** 32 - 1), (0, 5), (33, 1)])
@pytest.mark.parametrize("queries, keys", [(1, 500), (5, 500), (500, 500), (130, 450)])
def test_window_and_sinks(dev, dtype, window, sinks, queries, keys):
    dense(dev, np.random.default_rng(window % 1000 + sinks % 1000), dtype, 1, 2, 2, queries, keys, 32, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("queries", [1, 9, 140])
def test_lens_of_a_padded_batch(dev, dtype, causal, queries):
    # entries without keys, with fewer keys than queries, negative and beyond the end
    dense(dev, np.random.default_rng(queries), dtype, 7, 4, 2, queries, 150, 48, causal=causal, lens=[0, 1, 5, 149, 150, 1000, -3])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 4, 200])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_hidden_places_hold_does_not_matter(dev, dtype, queries, bad):
    def change(q, k, v):
        k[:, :, 170:], v[:, :, 170:] = bad, bad                # beyond lens
        k[0, :, 3] = bad                                       # behind the window of all queries but the first ones
        v[0, :, 3] = bad

    rng = np.random.default_rng(5)
    # hidden for every query: the rows behind lens, and key 3 where the window has passed it
    if queries == 200:
        dense(dev, rng, dtype, 1, 2, 1, 160, 200, 64, lens=[170], window=6, sinks=0, change=change)
    else:
        dense(dev, rng, dtype, 1, 2, 1, queries, 200, 64, lens=[170], window=50, sinks=2, change=change)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("queries, keys", [(150, 150), (40, 150)])
def test_a_value_that_some_rows_of_a_tile_see(dev, dtype, bad, queries, keys):
    """a NaN or an infinity among the values reaches the rows that see it, and no other row of its tile"""
    def change(q, k, v):
        v[:, :, 120, ::3] = bad

    rng = np.random.default_rng(6)
    for window, sinks in ((0, 0), (9, 2)):
        q, k, v = (ref.rounded(rng.standard_normal(s), dtype) for s in ((1, 2, queries, 64), (1, 1, keys, 64), (1, 1, keys, 64)))
        change(q, k, v)
        out = ref.values(dev.attention(*(ref.upload(dev, x, dtype) for x in (q, k, v)), window=window, sinks=sinks).to_numpy(), dtype)
        see = ref.visible(queries, keys, keys - queries, True, window, sinks)
        clean = np.where(np.isfinite(v), v, 0.0)
        for h in range(2):
            o, _, _, off, _, _ = ref.head(q[0, h], k[0, 0], clean[0, 0], see, 64 ** -0.5, dtype)
            o[np.ix_(see[:, 120], np.arange(64) % 3 == 0)] = bad
            ref.check(out[0, h], o, off, (window, h))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 33, 150])
def test_scores_that_differ_widely(dev, dtype, queries):
    """maxima that rise from tile to tile and weights that vanish against them"""
    def change(q, k, v):
        q[:], k[:] = np.abs(q), np.abs(k) * (np.arange(k.shape[2])[:, None] / 40)
        k[:] = ref.rounded(k, dtype)

    dense(dev, np.random.default_rng(7), dtype, 1, 2, 1, queries, 300, 64, change=change, causal=False)
    dense(dev, np.random.default_rng(8), dtype, 1, 2, 1, queries, 300, 64, scale=-3.0)
    dense(dev, np.random.default_rng(9), dtype, 1, 2, 1, queries, 300, 64, scale=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries, dim, pad", [(1, 64, 0), (70, 80, 0), (70, 64, 1), (5, 128, 3)])
def test_windows_of_one_projection(dev, dtype, queries, dim, pad):
    """q, k and v side by side in one buffer, rows of any pitch, and the result tokens first"""
    rng = np.random.default_rng(queries + dim)
    b, h, g = 2, 4, 2
    width = (h + 2 * g) * dim + pad
    rows = ref.rounded(rng.standard_normal((b, queries, width)), dtype)
    buf, strides = ref.upload(dev, rows, dtype), (queries * width, dim, width, 1)
    at = [0, h * dim, (h + g) * dim]
    q, k, v = (buf.view(o, (b, n, queries, dim)) if o + b * n * queries * dim <= rows.size else None for o, n in zip(at, (h, g, g)))
    out = dev.empty((b, h, queries, dim), q.dt)
    dev.attention(q, k, v, q_strides=strides, k_strides=strides, v_strides=strides, out=out, out_strides=(queries * h * dim, dim, h * dim, 1))
    got = ref.values(out.to_numpy(), dtype).reshape(b, queries, h, dim)
    x = rows[:, :, :(h + 2 * g) * dim].reshape(b, queries, h + 2 * g, dim)
    see = ref.visible(queries, queries, 0, True, 0, 0)
    for i in range(b):
        for j in range(h):
            o, _, _, off, _, _ = ref.head(x[i, :, j], x[i, :, h + j // 2], x[i, :, h + g + j // 2], see, dim ** -0.5, dtype)
            ref.check(got[i, :, j], o, off, (i, j))


@pytest.mark.parametrize("dtype", DTYPES)
def test_addresses_off_the_vector_grid(dev, dtype):
    rng = np.random.default_rng(11)
    for queries in (1, 40):
        x = [ref.rounded(rng.standard_normal((1, 2, n, 64)), dtype) for n in (queries, 90, 90)]
        bufs = [ref.upload(dev, np.concatenate([np.zeros(1), t.ravel()]), dtype).view(1, t.shape) for t in x]
        out = dev.empty((2 * queries * 64 + 1,), bufs[0].dt).view(1, x[0].shape)
        dev.attention(*bufs, out=out)
        got = ref.values(out.to_numpy(), dtype)
        for h in range(2):
            o, _, _, off, _, _ = ref.head(x[0][0, h], x[1][0, h], x[2][0, h], ref.visible(queries, 90, 90 - queries, True, 0, 0), 0.125, dtype)
            ref.check(got[0, h], o, off, h)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_key_shared_by_all_positions(dev, dtype):
    """strides of zero: one key and value row broadcast over the positions"""
    rng = np.random.default_rng(12)
    q, k, v = (ref.rounded(rng.standard_normal(s), dtype) for s in ((1, 2, 40, 64), (1, 2, 1, 64), (1, 2, 1, 64)))
    bufs = [ref.upload(dev, x, dtype) for x in (q, k, v)]
    wide = [b.reshape((1, 2, 1, 64)) for b in bufs[1:]]
    for b in wide:
        b.shape = (1, 2, 50, 64)
    got = ref.values(dev.attention(bufs[0], wide[0], wide[1], k_strides=(0, 64, 0, 1), v_strides=(0, 64, 0, 1)).to_numpy(), dtype)
    for h in range(2):
        kk, vv = np.repeat(k[0, h], 50, 0), np.repeat(v[0, h], 50, 0)
        o, _, _, off, _, _ = ref.head(q[0, h], kk, vv, ref.visible(40, 50, 10, True, 0, 0), 0.125, dtype)
        ref.check(got[0, h], o, off, h)


# ------------------------------------------------------------------------------------------------------------- paged
def paged(dev, p, window=0, sinks=0, scale=None, weights=None, lse=True, alias=False):
    """runs the problem and compares everything it may and may not touch"""
    scale = p.dim ** -0.5 if scale is None else scale
    cache = dev.paged_cache(ref.upload(dev, p.k, p.dtype), ref.upload(dev, p.v, p.dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    untouched = np.full(p.q.shape, 7.0)
    out, got_lse = ref.upload(dev, untouched, p.dtype), dev.upload(np.full(p.q.shape[:2], 7.0, np.float32)) if lse else None
    extra = {}
    if weights is not None:
        extra = {"weights": dev.upload(weights)}
        extra["weights_out"] = extra["weights"] if alias else dev.upload(np.where(np.isnan(weights), 7.0, weights).astype(np.float32))
    dev.paged_attention(ref.upload(dev, p.q, p.dtype), cache, dev.upload(p.starts_given if hasattr(p, "starts_given") else p.starts), window=window, sinks=sinks, scale=scale,
                        out=out, lse=got_lse, **extra)
    o, want_lse, received, o_off, lse_off, r_off = p.attention(scale, window, sinks, weights)
    left = np.zeros(o.shape, bool)
    left[:p.starts[0]] = left[p.starts[-1]:] = True
    got = ref.values(out.to_numpy(), p.dtype)
    assert (got[left] == 7.0).all(), "rows of no sequence were written"
    ref.check(got[~left], o[~left], o_off[~left], "o")
    if lse:
        ref.check(got_lse.to_numpy()[~left[..., 0]], want_lse[~left[..., 0]], lse_off[~left[..., 0]], "lse")
    if weights is not None:
        there = np.arange(p.cap)[None, None, :] < np.clip(p.lens, 0, p.cap)[:, None, None] + np.zeros((1, p.kv_heads, 1), int)
        w = extra["weights_out"].to_numpy()
        ref.check(w[there], received[there], r_off[there], "weights")
        before = weights if alias else np.where(np.isnan(weights), 7.0, weights).astype(np.float32)
        assert np.array_equal(w[~there], before[~there], equal_nan=True), "weights beyond the sequences were written"
    return cache, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 200])
@pytest.mark.parametrize("new", ["one", "chunks", "mixed"])
def test_pages(dev, dtype, page, new):
    rng = np.random.default_rng(page)
    lens = np.array([1, 64, 65, 190, 333, 40])
    count = {"one": np.ones(6, int), "chunks": np.array([1, 64, 20, 100, 333, 39]), "mixed": np.array([1, 1, 30, 1, 70, 1])}[new]
    paged(dev, ref.Paged(rng, dtype, 4, 2, 64, page, lens, count))
    paged(dev, ref.Paged(rng, dtype, 4, 2, 64, page, lens, count), window=50, sinks=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 4, 80), (8, 2, 128), (16, 1, 96), (34, 2, 40), (3, 1, 20), (2, 2, 256), (2, 1, 512), (40, 1, 64)])
def test_paged_head_layouts(dev, dtype, heads, kv_heads, dim):
    rng = np.random.default_rng(dim)
    for new in ([1, 1, 1], [3, 1, 150]):
        p = ref.Paged(rng, dtype, heads, kv_heads, dim, 16, [100, 1, 301], new)
        paged(dev, p, weights=rng.random((3, kv_heads, p.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 16, 32, 48, 56, 72, 104, 120, 136, 160, 192, 200, 248, 256])
def test_whole_vectors_of_columns(dev, dtype, dim):
    """every number of columns that the tiles take rows of, in chunks that end anywhere in a step"""
    rng = np.random.default_rng(dim)
    dense(dev, rng, dtype, 2, 4, 2, 150, 333, dim, lens=[333, 170])
    dense(dev, rng, dtype, 1, 2, 2, 200, 200, dim, window=70, sinks=3)
    for new in ([1, 1, 1], [70, 2, 140]):
        p = ref.Paged(rng, dtype, 4, 2, dim, 24, [100, 9, 301], new)
        paged(dev, p, weights=rng.random((3, 2, p.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window, sinks", [(0, 0), (40, 0), (40, 5), (3, 90)])
@pytest.mark.parametrize("alias", [False, True])
def test_received_weights(dev, dtype, window, sinks, alias):
    """old tokens add to what they had, new ones start from nothing, whatever stood there before"""
    rng = np.random.default_rng(window + sinks)
    for new in ([1, 1, 1, 0, 1], [17, 130, 1, 0, 4]):
        p = ref.Paged(rng, dtype, 4, 2, 64, 16, [17, 200, 90, 33, 4], new)
        w = rng.random((5, 2, p.cap), dtype=np.float32)
        for b in range(5):
            w[b, :, p.lens[b] - new[b]:] = np.nan              # new tokens' places, and those beyond
        paged(dev, p, window=window, sinks=sinks, weights=w, lse=bool(alias), alias=alias)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("most", [1, 90])
def test_sequences_without_keys_rows_or_pages(dev, dtype, most):
    rng = np.random.default_rng(most)
    # no keys; no new tokens; more new tokens than keys; a page missing in front, in the middle, at the end; all pages missing; lens beyond the table
    lens = np.array([0, 50, 3, 120, 120, 120, 40, 31])
    new = np.array([2, 0, 5, most, most, most, min(most, 40), min(most, 31)])
    p = ref.Paged(rng, dtype, 4, 2, 64, 16, lens, new, holes=[(3, 0), (4, 3), (5, 7), (6, 0), (6, 1), (6, 2)])
    paged(dev, p, weights=rng.random((8, 2, p.cap), dtype=np.float32))
    paged(dev, p, window=20, sinks=2, weights=rng.random((8, 2, p.cap), dtype=np.float32))
    long = ref.Paged(rng, dtype, 4, 2, 64, 16, np.array([60, 20]), np.array([1, 3]), spare=0)
    long.lens = np.array([70, -5])                             # six tokens more than there is room for; fewer than none
    paged(dev, long, weights=rng.random((2, 2, long.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_no_sequence_stay_as_they_were(dev, dtype):
    rng = np.random.default_rng(3)
    for new in ([1, 1, 1], [40, 1, 7]):
        p = ref.Paged(rng, dtype, 4, 2, 64, 16, [100, 20, 57], new)
        extra = ref.rounded(rng.standard_normal((9, 4, 64)), dtype)
        p.q = np.concatenate([extra[:4], p.q, extra[4:]])
        p.starts = p.starts + 4
        p.tokens = p.q.shape[0]
        paged(dev, p, weights=rng.random((3, 2, p.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_starts_outside_of_the_tokens_are_taken_into_them(dev, dtype):
    rng = np.random.default_rng(4)
    p = ref.Paged(rng, dtype, 4, 2, 64, 16, [100, 20, 57], [3, 1, 2])
    p.starts_given = p.starts.copy()
    p.starts_given[0], p.starts_given[-1] = -5, 1000           # the first and last sequence's rows end with the tokens
    paged(dev, p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqs", [64, 65, 300])
def test_many_sequences(dev, dtype, seqs):
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, 60, seqs)
    new = np.minimum(rng.integers(0, 4, seqs), lens)
    p = ref.Paged(rng, dtype, 2, 1, 32, 8, lens, new)
    paged(dev, p, weights=rng.random((seqs, 1, p.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 60, 700])
def test_long_caches(dev, dtype, new):
    """one long sequence among short ones: its keys are split over the chip"""
    rng = np.random.default_rng(new)
    p = ref.Paged(rng, dtype, 4, 1, 64, 32, [9000, 100, 5000], [new, 1, 1])
    paged(dev, p, weights=rng.random((3, 1, p.cap), dtype=np.float32))
    paged(dev, p, window=4000, sinks=10)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 80])
def test_stale_rows_of_pages_do_not_matter(dev, dtype, new):
    """what the cache's pages hold behind the last token and in pages of nobody may be anything"""
    rng = np.random.default_rng(new)
    p = ref.Paged(rng, dtype, 4, 2, 64, 16, [100, 83], [new, min(new, 83)])
    used = np.zeros((p.pages, 16), bool)
    for b, n in enumerate(p.lens):
        t = np.arange(n)
        used[p.table[b, t // 16], t % 16] = True
    p.k[np.broadcast_to(~used[:, None, :, None], p.k.shape)] = np.nan
    p.v[np.broadcast_to(~used[:, None, :, None], p.v.shape)] = np.inf
    paged(dev, p, weights=rng.random((2, 2, p.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_shared_pages_and_strided_rows(dev, dtype):
    """two sequences with one prefix, queries as a window of a projection"""
    rng = np.random.default_rng(14)
    p = ref.Paged(rng, dtype, 4, 2, 64, 16, [100, 77], [1, 20])
    p.table[1, :3] = p.table[0, :3]
    rows = rng.standard_normal((p.tokens, 8, 64))
    rows[:, :4] = p.q
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    q = ref.upload(dev, rows, dtype).view(0, (p.tokens, 4, 64))
    got = ref.values(dev.paged_attention(q, cache, dev.upload(p.starts), q_strides=(8 * 64, 64)).to_numpy(), dtype)
    o, _, _, off, _, _ = p.attention(0.125)
    ref.check(got, o, off, "o")


# ------------------------------------------------------------------------------------------------- together, recorded
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("recorded", [False, True])
def test_a_conversation(dev, dtype, recorded):
    """prompt in, tokens one by one, cut, tokens again: append, attention and eviction together as a serving loop makes them"""
    from test_gpu_paged import host_append, host_evict

    rng = np.random.default_rng(21)
    heads, g, d, page, keep = 4, 2, 64, 16, 40
    p = ref.Paged(rng, dtype, heads, g, d, page, [70, 30], [70, 30], spare=3)
    for b in range(2):                                         # room for what will come
        p.table[b, p.table[b] < 0] = -1
    fresh = iter(p.free)
    for b, i in ((0, int(np.sum(p.table[0] >= 0))), (1, int(np.sum(p.table[1] >= 0)))):
        p.table[b, i] = next(fresh)
    k_dev, v_dev, table, lens = ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32))
    cache = dev.paged_cache(k_dev, v_dev, table, lens)
    weights = np.zeros((2, g, p.cap), np.float32)
    w_dev = dev.upload(weights)
    received_off = np.zeros(weights.shape)
    graph = None
    for step in range(7):
        new = [70, 30] if step == 0 else [1, 1]
        if step:
            p.lens = p.lens + 1
            from_host = p.lens.astype(np.int32)
            lens.device.lib.rt_h2d(dev.handle, lens.ptr, from_host.ctypes.data, from_host.nbytes)
        p.new, p.starts = np.array(new), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        p.tokens = int(sum(new))
        rows = ref.rounded(rng.standard_normal((p.tokens, heads + 2 * g, d)), dtype)
        p.q = rows[:, :heads]
        host_append(p, rows[:, heads:heads + g], rows[:, heads + g:])
        strides = ((heads + 2 * g) * d, d)
        if step < 2 or not recorded:
            buf, starts = ref.upload(dev, rows, dtype), dev.upload(p.starts)
            out, q = dev.empty((p.tokens, heads, d), buf.dt), buf.view(0, (p.tokens, heads, d))
            kk, vv = buf.view(heads * d, (p.tokens, g, d)), buf.view((heads + g) * d, (p.tokens, g, d))

        def work():
            dev.paged_append(cache, starts, kk, vv, k_strides=strides, v_strides=strides)
            dev.paged_attention(q, cache, starts, out=out, q_strides=strides, weights=w_dev)

        if recorded and step:
            if graph is None:                                  # recorded once, replayed on what the buffers then hold
                with dev.capture() as graph:
                    work()
            else:
                a = ref.raw(rows, dtype)
                dev.lib.rt_h2d(dev.handle, buf.ptr, a.ctypes.data, a.nbytes)
            graph.launch()
        else:
            work()
        o, _, received, o_off, _, r_off = p.attention(d ** -0.5, weights=weights)
        ref.check(ref.values(out.to_numpy(), dtype), o, o_off, ("o", step))
        there = np.arange(p.cap)[None, None] < p.lens[:, None, None] + np.zeros((1, g, 1), int)
        got = w_dev.to_numpy()
        received_off = np.where(there, received_off + r_off, 0.0)
        ref.check(got[there], received[there], received_off[there], ("weights", step))
        weights = got                                          # the next step starts from what the device has
        received_off[:] = 0.0
        if step in (0, 3):
            dev.paged_evict(cache, w_dev, keep, first=2, recent=8)
            host_evict(p, weights, keep, 2, 8)
            assert np.array_equal(lens.to_numpy(), p.lens), step
            assert np.array_equal(ref.values(k_dev.to_numpy(), dtype), p.k) and np.array_equal(ref.values(v_dev.to_numpy(), dtype), p.v), step
            weights = w_dev.to_numpy()


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_graphs_and_eager_calls_share_the_workspace(dev, dtype):
    """graphs of different sizes replayed in turn with eager calls between them, each result as its eager one"""
    rng = np.random.default_rng(31)
    runs = []
    for lens, new in (([5000, 70], [1, 1]), ([300, 900, 40], [1, 60, 1])):
        p = ref.Paged(rng, dtype, 4, 2, 64, 16, lens, new)
        cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
        q, starts, w = ref.upload(dev, p.q, dtype), dev.upload(p.starts), dev.upload(rng.random((len(lens), 2, p.cap), dtype=np.float32))
        w_out, out = dev.upload(np.zeros(w.shape, np.float32)), dev.empty(p.q.shape, q.dt)

        def work(q=q, cache=cache, starts=starts, out=out, w=w, w_out=w_out):
            dev.paged_attention(q, cache, starts, out=out, weights=w, weights_out=w_out)

        work()
        runs.append((work, out, w_out, out.to_numpy(), w_out.to_numpy()))
    graphs = []
    for work, *_ in runs:
        with dev.capture() as g:
            work()
        graphs.append(g)
    # an eager call that outgrows the workspace the graphs were recorded with
    big = ref.Paged(rng, dtype, 16, 2, 64, 16, [3000] * 12, [1] * 12)
    paged(dev, big, weights=rng.random((12, 2, big.cap), dtype=np.float32))
    for _ in range(3):
        for i, (work, out, w_out, want, want_w) in enumerate(runs):
            out.zero_()
            w_out.zero_()
            graphs[i].launch()
            graphs[1 - i].launch()
            assert np.array_equal(out.to_numpy().view(np.uint8), want.view(np.uint8)) and np.array_equal(w_out.to_numpy(), want_w), i
            runs[1 - i][0]()
            dev.sync()


def test_a_graph_with_attention_stays_on_its_device():
    """another rt_device of the same GPU has another workspace and another stream: refused there"""
    from ratchet_amd import Device, RatchetError

    a, b = Device(0), Device(0)
    rng = np.random.default_rng(1)
    p = ref.Paged(rng, "f16", 4, 2, 64, 16, [700], [1])
    cache = a.paged_cache(ref.upload(a, p.k, "f16"), ref.upload(a, p.v, "f16"), a.upload(p.table), a.upload(p.lens.astype(np.int32)))
    q, starts, w = ref.upload(a, p.q, "f16"), a.upload(p.starts), a.upload(np.zeros((1, 2, p.cap), np.float32))
    out = a.empty(p.q.shape, q.dt)
    a.paged_attention(q, cache, starts, out=out, weights=w)
    with a.capture() as g:
        a.paged_attention(q, cache, starts, out=out, weights=w)
    g.launch()
    a.sync()
    assert b.lib.rt_graph_launch(b.handle, g.graph.handle) == 7                # RT_ERR_ARG
    b.close()
    g.graph = None
    a.close()


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_call_gives_the_same_bits(dev, dtype):
    rng = np.random.default_rng(41)
    p = ref.Paged(rng, dtype, 8, 2, 128, 16, [4000, 900, 12], [1, 300, 1])
    w = rng.random((3, 2, p.cap), dtype=np.float32)
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    q, starts, w_in = ref.upload(dev, p.q, dtype), dev.upload(p.starts), dev.upload(w)
    seen = []
    for _ in range(4):
        w_out = dev.upload(np.zeros(w.shape, np.float32))
        out = dev.paged_attention(q, cache, starts, weights=w_in, weights_out=w_out)
        seen.append(out.to_numpy().tobytes() + w_out.to_numpy().tobytes())
    assert len(set(seen)) == 1


# ---------------------------------------------------------------------------------------------------- large and odd
@pytest.mark.parametrize("queries", [1, 70])
def test_keys_beyond_4_gib(dev, queries):
    """2^25 keys of 128 bytes; a window over the last ones and two sinks at the other end"""
    rng = np.random.default_rng(queries)
    keys, window = 1 << 25, 500
    k, v = dev.empty((1, 1, keys, 64), _lib.F16), dev.empty((1, 1, keys, 64), _lib.F16)
    tail = window + queries
    rows = {}
    for name, buf in (("k", k), ("v", v)):
        first, last = ref.rounded(rng.standard_normal((2, 64)), "f16"), ref.rounded(rng.standard_normal((tail, 64)), "f16")
        buf.view(0, (2, 64)).upload(ref.raw(first, "f16"))
        buf.view((keys - tail) * 64, (tail, 64)).upload(ref.raw(last, "f16"))
        rows[name] = np.concatenate([first, last])
    q = ref.rounded(rng.standard_normal((1, 1, queries, 64)), "f16")
    got = ref.values(dev.attention(ref.upload(dev, q, "f16"), k, v, window=window, sinks=2).to_numpy(), "f16")
    p, t = np.arange(queries)[:, None] + keys - queries, np.concatenate([np.arange(2), np.arange(keys - tail, keys)])[None, :]
    o, _, _, off, _, _ = ref.head(q[0, 0], rows["k"], rows["v"], (t <= p) & ((p - t < window) | (t < 2)), 0.125, "f16")
    ref.check(got[0, 0], o, off, "o")


@pytest.mark.parametrize("new", [[1, 1], [1, 200]])
def test_pages_beyond_4_gib(dev, new):
    """append, attention, received weights and eviction on pages on either side of byte 2^32 of the pools"""
    from test_gpu_paged import host_append, host_evict

    rng = np.random.default_rng(sum(new))
    p = ref.Paged(rng, "f16", 4, 2, 64, 32, [400, 300], new, spare=1)
    per = 2 * 32 * 64                                          # elements of a page
    pages = (1 << 32) // (2 * per) + 40
    where = np.sort(rng.choice(np.concatenate([np.arange(20), np.arange(pages - 60, pages)]), p.pages, replace=False))
    kb, vb = dev.empty((pages, 2, 32, 64), _lib.F16), dev.empty((pages, 2, 32, 64), _lib.F16)
    for i, at in enumerate(where):
        kb.view(int(at) * per, (per,)).upload(ref.raw(p.k[i], "f16").ravel())
        vb.view(int(at) * per, (per,)).upload(ref.raw(p.v[i], "f16").ravel())
    table = np.where(p.table >= 0, where[np.maximum(p.table, 0)], -1).astype(np.int32)
    cache = dev.paged_cache(kb, vb, dev.upload(table), dev.upload(p.lens.astype(np.int32)))
    k, v = (ref.rounded(rng.standard_normal((p.tokens, 2, 64)), "f16") for _ in range(2))
    starts, w = dev.upload(p.starts), rng.random((2, 2, p.cap), dtype=np.float32)
    w_dev = dev.upload(w)
    dev.paged_append(cache, starts, ref.upload(dev, k, "f16"), ref.upload(dev, v, "f16"))
    host_append(p, k, v)
    got = ref.values(dev.paged_attention(ref.upload(dev, p.q, "f16"), cache, starts, weights=w_dev).to_numpy(), "f16")
    o, _, received, off, _, r_off = p.attention(0.125, weights=w)
    ref.check(got, o, off, "o")
    there = np.arange(p.cap)[None, None] < p.lens[:, None, None] + np.zeros((1, 2, 1), int)
    now = w_dev.to_numpy()
    ref.check(now[there], received[there], r_off[there], "weights")
    dev.paged_evict(cache, w_dev, 100, first=4, recent=20)
    host_evict(p, now, 100, 4, 20)
    for i, at in enumerate(where):
        assert np.array_equal(ref.values(kb.view(int(at) * per, (2, 32, 64)).to_numpy(), "f16"), p.k[i]), i
        assert np.array_equal(ref.values(vb.view(int(at) * per, (2, 32, 64)).to_numpy(), "f16"), p.v[i]), i


@pytest.mark.parametrize("seqs, cap_pages", [(200, 300), (3, 40000)])
def test_more_room_than_blocks(dev, seqs, cap_pages):
    """weights of chunks where the table has room for far more keys than there are"""
    rng = np.random.default_rng(seqs)
    lens = rng.integers(1, 300, seqs)
    p = ref.Paged(rng, "f16", 2, 1, 32, 16, lens, np.minimum(rng.integers(10, 60, seqs), lens), spare=cap_pages)
    paged(dev, p, weights=rng.random((seqs, 1, p.cap), dtype=np.float32))


def test_many_ragged_chunks(dev):
    """row tiles of many lengths, whose pieces add up to the most that a launch has room for"""
    for seed in range(4):
        rng = np.random.default_rng(seed)
        lens = rng.integers(1, 1500, 20)
        new = np.maximum(1, (lens * rng.random(20) ** 2).astype(int))
        paged(dev, ref.Paged(rng, "bf16", 4, 2, 64, 16, lens, new))
    rng = np.random.default_rng(9)
    lens = np.array([9000] + [300] * 12)                        # one long walk among short ones
    paged(dev, ref.Paged(rng, "bf16", 8, 1, 64, 16, lens, [140] + [129] * 12))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("batch, heads, kv_heads, queries, keys, lens", [(1, 64, 64, 512, 512, None), (3, 33, 11, 130, 700, [700, 5, 333]), (1, 300, 300, 129, 200, None),
                                                                         (1, 32, 32, 1030, 1030, None), (1, 64, 16, 260, 2900, None)])
def test_row_tiles_that_fill_the_chip(dev, dtype, causal, batch, heads, kv_heads, queries, keys, lens):
    """256 row tiles and more: a block to each, in rounds that pair long walks with short ones, or shared out where the walks are long"""
    dense(dev, np.random.default_rng(heads), dtype, batch, heads, kv_heads, queries, keys, 32, causal=causal, lens=lens)


@pytest.mark.parametrize("queries", [1, 140])
@pytest.mark.parametrize("window", [1 << 30, (1 << 31) - 2, 1 << 31])
def test_windows_wider_than_any_position(dev, queries, window):
    dense(dev, np.random.default_rng(1), "f16", 1, 2, 1, queries, 100, 64, window=window, sinks=1)


def test_lens_far_beyond_the_table(dev):
    """tokens that there is no room for: the queries sit behind all keys, and a window has passed those that are there"""
    rng = np.random.default_rng(2)
    for window, sinks in ((0, 0), (10, 0), (10, 3)):
        p = ref.Paged(rng, "f16", 4, 2, 64, 16, np.array([60, 20]), np.array([1, 40]), spare=0)
        p.lens = np.array([(1 << 30) - 1, 1000])
        paged(dev, p, window=window, sinks=sinks, weights=rng.random((2, 2, p.cap), dtype=np.float32))


def test_two_devices_at_once():
    """two rt_devices of one GPU have their own streams and workspaces: calls that overlap do not meet"""
    from ratchet_amd import Device

    devs = [Device(0), Device(0)]
    rng = np.random.default_rng(3)
    runs = []
    for d in devs:
        p = ref.Paged(rng, "bf16", 8, 2, 128, 16, [3000, 900, 12], [1, 1, 1])
        w = rng.random((3, 2, p.cap), dtype=np.float32)
        cache = d.paged_cache(ref.upload(d, p.k, "bf16"), ref.upload(d, p.v, "bf16"), d.upload(p.table), d.upload(p.lens.astype(np.int32)))
        args = ref.upload(d, p.q, "bf16"), cache, d.upload(p.starts)
        out, w_in, w_out = d.empty(p.q.shape, _lib.BF16), d.upload(w), d.upload(np.zeros_like(w))
        d.paged_attention(*args, out=out, weights=w_in, weights_out=w_out)
        runs.append((d, args, out, w_in, w_out, out.to_numpy(), w_out.to_numpy()))
    for _ in range(20):
        for d, args, out, w_in, w_out, *_ in runs:
            d.paged_attention(*args, out=out, weights=w_in, weights_out=w_out)
    for d, _, out, _, w_out, want, want_w in runs:
        assert np.array_equal(out.to_numpy(), want) and np.array_equal(w_out.to_numpy(), want_w)
    for d in devs:
        d.close()
