"""Attention where a call's parts differ: rows that the matrix-unit tiles cannot take, under every mask, and long pieces of a prompt next to many
single tokens.  Against the definitions in 64 bits, within the bounds of attention_ref.py."""
import numpy as np
import pytest

import attention_ref as ref
from test_gpu_attention import DTYPES, dense, paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ratchet_amd import Device

    d = Device(0)
    yield d
    d.close()


# ------------------------------------------------------------------------------- 7 columns are no whole vectors in any type, 264 are beyond the tiles
ODD = [7, 264]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", ODD)
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (7, 3), (64, 64), (65, 4), (100, 130), (1000, 4), (2 ** 32 - 1, 2 ** 32 - 1)])
@pytest.mark.parametrize("queries, keys", [(1, 400), (5, 400), (150, 150), (130, 350)])
def test_window_and_sinks(dev, dtype, dim, window, sinks, queries, keys):
    dense(dev, np.random.default_rng(window % 1000 + sinks % 1000), dtype, 1, 2, 2, queries, keys, dim, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", ODD)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("queries", [1, 9, 140])
def test_lens_of_a_padded_batch(dev, dtype, dim, causal, queries):
    dense(dev, np.random.default_rng(queries), dtype, 7, 4, 2, queries, 150, dim, causal=causal, lens=[0, 1, 5, 149, 150, 1000, -3])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", ODD)
@pytest.mark.parametrize("queries", [1, 4, 160])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_hidden_places_hold_does_not_matter(dev, dtype, dim, queries, bad):
    def change(q, k, v):
        k[:, :, 170:], v[:, :, 170:] = bad, bad                # beyond lens
        k[0, :, 3], v[0, :, 3] = bad, bad                      # behind every query's window

    dense(dev, np.random.default_rng(5), dtype, 1, 2, 1, queries, 200, dim, lens=[170], window=6 if queries == 160 else 50, sinks=0 if queries == 160 else 2, change=change)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", ODD)
def test_scores_that_differ_widely(dev, dtype, dim):
    def change(q, k, v):
        q[:], k[:] = np.abs(q), ref.rounded(np.abs(k) * (np.arange(k.shape[2])[:, None] / 40), dtype)

    for queries in (1, 150):
        dense(dev, np.random.default_rng(7), dtype, 1, 2, 1, queries, 300, dim, change=change, causal=False)
        dense(dev, np.random.default_rng(8), dtype, 1, 2, 1, queries, 300, dim, scale=-3.0)
        dense(dev, np.random.default_rng(9), dtype, 1, 2, 1, queries, 300, dim, scale=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", ODD)
@pytest.mark.parametrize("window, sinks", [(0, 0), (40, 0), (40, 5), (3, 90)])
@pytest.mark.parametrize("alias", [False, True])
def test_received_weights(dev, dtype, dim, window, sinks, alias):
    rng = np.random.default_rng(window + sinks)
    for new in ([1, 1, 1, 0, 1], [17, 130, 1, 0, 4]):
        p = ref.Paged(rng, dtype, 4, 2, dim, 16, [17, 200, 90, 33, 4], new)
        w = rng.random((5, 2, p.cap), dtype=np.float32)
        for b in range(5):
            w[b, :, p.lens[b] - new[b]:] = np.nan
        paged(dev, p, window=window, sinks=sinks, weights=w, lse=bool(alias), alias=alias)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", ODD)
@pytest.mark.parametrize("most", [1, 90])
def test_sequences_without_keys_rows_or_pages(dev, dtype, dim, most):
    rng = np.random.default_rng(most)
    lens = np.array([0, 50, 3, 120, 120, 120, 40, 31])
    new = np.array([2, 0, 5, most, most, most, min(most, 40), min(most, 31)])
    p = ref.Paged(rng, dtype, 4, 2, dim, 16, lens, new, holes=[(3, 0), (4, 3), (5, 7), (6, 0), (6, 1), (6, 2)])
    paged(dev, p, weights=rng.random((8, 2, p.cap), dtype=np.float32))
    paged(dev, p, window=20, sinks=2, weights=rng.random((8, 2, p.cap), dtype=np.float32))
    long = ref.Paged(rng, dtype, 4, 2, dim, 16, np.array([60, 20]), np.array([1, 3]), spare=0)
    long.lens = np.array([70, -5])
    paged(dev, long, weights=rng.random((2, 2, long.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", ODD)
def test_rows_of_no_sequence_and_starts_outside(dev, dtype, dim):
    rng = np.random.default_rng(3)
    for new in ([1, 1, 1], [40, 1, 7]):
        p = ref.Paged(rng, dtype, 4, 2, dim, 16, [100, 20, 57], new)
        extra = ref.rounded(rng.standard_normal((9, 4, dim)), dtype)
        p.q = np.concatenate([extra[:4], p.q, extra[4:]])
        p.starts = p.starts + 4
        p.tokens = p.q.shape[0]
        paged(dev, p, weights=rng.random((3, 2, p.cap), dtype=np.float32))
    p = ref.Paged(rng, dtype, 4, 2, dim, 16, [100, 20, 57], [3, 1, 2])
    p.starts_given = p.starts.copy()
    p.starts_given[0], p.starts_given[-1] = -5, 1000
    paged(dev, p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqs", [64, 65, 300])
def test_many_sequences(dev, dtype, seqs):
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, 60, seqs)
    new = np.minimum(rng.integers(0, 4, seqs), lens)
    p = ref.Paged(rng, dtype, 2, 1, 7, 8, lens, new)
    paged(dev, p, weights=rng.random((seqs, 1, p.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", ODD)
@pytest.mark.parametrize("new", [1, 80])
def test_stale_rows_of_pages_do_not_matter(dev, dtype, dim, new):
    rng = np.random.default_rng(new)
    p = ref.Paged(rng, dtype, 4, 2, dim, 16, [100, 83], [new, min(new, 83)])
    used = np.zeros((p.pages, 16), bool)
    for b, n in enumerate(p.lens):
        t = np.arange(n)
        used[p.table[b, t // 16], t % 16] = True
    p.k[np.broadcast_to(~used[:, None, :, None], p.k.shape)] = np.nan
    p.v[np.broadcast_to(~used[:, None, :, None], p.v.shape)] = np.inf
    paged(dev, p, weights=rng.random((2, 2, p.cap), dtype=np.float32))


# ------------------------------------------------------------------------------------------- pieces of a prompt next to many single tokens
def serving_step(rng, dtype, heads, kv_heads, dim, seqs, chunk, longest, page=32):
    """one sequence brings `chunk` tokens and has `longest` keys, the others one token each: few rows a sequence on average"""
    lens = rng.integers(1, 250, seqs)
    lens[seqs // 2] = longest
    lens[3] = longest // 2
    new = np.ones(seqs, int)
    new[seqs // 2] = chunk
    assert new.sum() * (heads // kv_heads) <= 16 * seqs
    return ref.Paged(rng, dtype, heads, kv_heads, dim, page, lens, new)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, dim, chunk, longest", [(2, 2, 64, 700, 6000), (1, 1, 96, 300, 9000), (2, 2, 40, 17, 9000), (4, 1, 128, 150, 5000), (1, 1, 256, 129, 3000), (2, 2, 80, 128, 700)])
@pytest.mark.parametrize("weighed", [False, True])
def test_a_piece_of_a_prompt_among_tokens(dev, dtype, heads, kv_heads, dim, chunk, longest, weighed):
    rng = np.random.default_rng(chunk)
    p = serving_step(rng, dtype, heads, kv_heads, dim, 60, chunk, longest)
    weights = rng.random((60, kv_heads, p.cap), dtype=np.float32) if weighed else None
    paged(dev, p, weights=weights, lse=not weighed)
    paged(dev, p, window=longest // 3, sinks=5, weights=weights)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_piece_whose_scores_are_too_many_to_keep(dev, dtype):
    rng = np.random.default_rng(1)
    p = serving_step(rng, dtype, 8, 8, 32, 60, 800, 10000)
    assert p.tokens * 8 * p.cap * 4 > 256 << 20
    paged(dev, p, weights=rng.random((60, 8, p.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_value_that_some_rows_of_a_piece_see(dev, dtype, bad):
    """it reaches the rows that see it and no others, also where a row's keys are shared out over blocks"""
    rng = np.random.default_rng(2)
    p = serving_step(rng, dtype, 2, 2, 64, 60, 400, 5000)
    b, t, window = 30, 4500, 300
    o, _, _, off, _, _ = p.attention(0.125, window=window, sinks=3)
    p.v[p.table[b, t // p.page], :, t % p.page, ::3] = bad
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    got = ref.values(dev.paged_attention(ref.upload(dev, p.q, dtype), cache, dev.upload(p.starts), window=window, sinks=3, scale=0.125).to_numpy(), dtype)
    at = np.arange(400) + p.lens[b] - 400
    rows = p.starts[b] + np.flatnonzero((t <= at) & (at - t < window))
    assert 0 < len(rows) < 400
    o[rows[:, None, None], np.arange(2)[:, None], np.arange(64)[::3]] = bad
    ref.check(got, o, off, "o")


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_step_gives_the_same_bits(dev, dtype):
    rng = np.random.default_rng(4)
    p = serving_step(rng, dtype, 4, 2, 128, 60, 300, 6000)
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    q, starts, w = ref.upload(dev, p.q, dtype), dev.upload(p.starts), dev.upload(rng.random((60, 2, p.cap), dtype=np.float32))
    seen = set()
    for _ in range(4):
        w_out = dev.upload(np.zeros((60, 2, p.cap), np.float32))
        seen.add(dev.paged_attention(q, cache, starts, weights=w, weights_out=w_out).to_numpy().tobytes() + w_out.to_numpy().tobytes())
    assert len(seen) == 1
