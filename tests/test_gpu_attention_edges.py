"""Edges of attention: scores of minus infinity, lengths of a padded batch over many keys, strides of extents of one."""
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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [7, 40, 64, 80, 256])
@pytest.mark.parametrize("new", [[1, 1, 1], [90, 1, 200]])
def test_rows_whose_visible_scores_are_all_minus_infinity(dev, dtype, dim, new):
    """they weigh nothing, as keys out of sight do: a result of 0, an lse of -inf, and nothing received from them"""
    rng = np.random.default_rng(dim)
    p = ref.Paged(rng, dtype, 4, 2, dim, 16, [300, 80, 250], new)
    p.q[..., 0] = np.abs(p.q[..., 0]) + 1.0
    p.q = ref.rounded(p.q, dtype)
    t = np.arange(300)
    p.k[p.table[0, t // 16], :, t % 16, 0] = -np.inf            # all of sequence 0
    t = np.arange(0, 250, 3)
    p.k[p.table[2, t // 16], :, t % 16, 0] = -np.inf            # every third key of sequence 2
    w = rng.random((3, 2, p.cap), dtype=np.float32)
    lse, w_out = dev.upload(np.zeros(p.q.shape[:2], np.float32)), dev.upload(np.zeros(w.shape, np.float32))
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    out = dev.paged_attention(ref.upload(dev, p.q, dtype), cache, dev.upload(p.starts), scale=0.125, lse=lse, weights=dev.upload(w), weights_out=w_out)
    got, got_lse, got_w = ref.values(out.to_numpy(), dtype), lse.to_numpy(), w_out.to_numpy()
    for b in range(3):
        lo, hi, n = p.starts[b], p.starts[b + 1], int(p.lens[b])
        k, _ = p.rows(p.k, b)
        v, _ = p.rows(p.v, b)
        shift = n - (hi - lo)
        for g in range(2):
            total, off = np.where(np.arange(n) < shift, w[b, g, :n].astype(np.float64), 0.0), np.zeros(n)
            gone = np.isinf(k[g, :, 0])
            clean = np.where(gone[:, None], 0.0, k[g])
            see = ref.visible(hi - lo, n, shift, True, 0, 0, gone)
            for h in (2 * g, 2 * g + 1):
                o, want_lse, x, o_off, lse_off, factor = ref.head(p.q[lo:hi, h], clean, v[g], see, 0.125, dtype)
                ref.check(got[lo:hi, h], o, o_off, ("o", b, h))
                ref.check(got_lse[lo:hi, h], want_lse, lse_off, ("lse", b, h))
                total += x.sum(axis=0)
                off += (x * factor[:, None]).sum(axis=0)
            ref.check(got_w[b, g, :n], total, off + (2 * (hi - lo) + 1) * ref.U * np.abs(total), ("weights", b, g))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 104])
@pytest.mark.parametrize("causal, window, sinks", [(True, 0, 0), (True, 700, 0), (True, 700, 9), (False, 0, 0)])
@pytest.mark.parametrize("queries", [1, 16, 150])
def test_lens_of_a_padded_batch_over_many_keys(dev, dtype, dim, causal, window, sinks, queries):
    """entries whose keys are shared out over blocks next to those with none, and with fewer keys than queries"""
    dense(dev, np.random.default_rng(queries), dtype, 6, 2, 1, queries, 3000, dim, causal=causal, window=window, sinks=sinks, lens=[0, 1, 5, 2999, 3000, 1400])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries, keys, heads, kv_heads", [(1, 90, 4, 1), (40, 40, 1, 1), (1, 1, 2, 2)])
def test_strides_of_extents_of_one(dev, dtype, queries, keys, heads, kv_heads):
    """nothing is ever that far away, so they change nothing: the same bits"""
    rng = np.random.default_rng(keys)
    q, k, v = (ref.upload(dev, ref.rounded(rng.standard_normal(s), dtype), dtype) for s in ((1, heads, queries, 64), (1, kv_heads, keys, 64), (1, kv_heads, keys, 64)))

    def odd(shape):
        dense_strides = (shape[1] * shape[2] * 64, shape[2] * 64, 64, 1)
        return tuple(s if n > 1 else 7 + 2 * i for i, (n, s) in enumerate(zip(shape, dense_strides)))

    want = dev.attention(q, k, v).to_numpy()
    got = dev.attention(q, k, v, q_strides=odd(q.shape), k_strides=odd(k.shape), v_strides=odd(v.shape), out=dev.empty(q.shape, q.dt), out_strides=odd(q.shape)).to_numpy()
    assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    # one token, one KV head over pages
    p = ref.Paged(rng, dtype, 1, 1, 64, 16, [80], [1])
    cache = dev.paged_cache(ref.upload(dev, p.k, dtype), ref.upload(dev, p.v, dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    x, starts = ref.upload(dev, p.q, dtype), dev.upload(p.starts)
    want = dev.paged_attention(x, cache, starts).to_numpy()
    assert np.array_equal(dev.paged_attention(x, cache, starts, q_strides=(65, 67)).to_numpy().view(np.uint8), want.view(np.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [4, 12, 28, 60, 76, 100, 132, 252])
def test_whole_vectors_of_f32_columns(dev, dtype, dim):
    """a multiple of 4 is whole vectors in f32 and not in 16 bits; 4 columns are one"""
    rng = np.random.default_rng(dim)
    dense(dev, rng, dtype, 2, 4, 2, 140, 300, dim, lens=[300, 170])
    for new in ([1, 1, 1], [70, 2, 140]):
        p = ref.Paged(rng, dtype, 4, 2, dim, 24, [100, 9, 301], new)
        paged(dev, p, weights=rng.random((3, 2, p.cap), dtype=np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads", [(130, 1), (400, 2), (129, 3)])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 20]])
def test_more_heads_to_a_kv_head_than_rows_to_a_tile(dev, dtype, heads, kv_heads, new):
    rng = np.random.default_rng(heads)
    p = ref.Paged(rng, dtype, heads, kv_heads, 64, 16, [900, 33, 300], new)
    weights = rng.random((3, kv_heads, p.cap), dtype=np.float32)
    paged(dev, p, weights=weights)
    paged(dev, p, window=100, sinks=3, weights=weights)
    dense(dev, rng, dtype, 2, heads, kv_heads, new[0], 200, 64, lens=[200, 5])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, new", [(8, 2, [1] * 5), (6, 2, [1, 90, 7, 1, 33]), (32, 4, [2, 1, 1, 300, 1])])
@pytest.mark.parametrize("window, sinks", [(1, 0), (17, 40), (64, 1), (129, 0), (500, 200)])
def test_windows_of_shared_heads_over_pages(dev, dtype, heads, kv_heads, new, window, sinks):
    rng = np.random.default_rng(window)
    p = ref.Paged(rng, dtype, heads, kv_heads, 48, 24, [1500, 400, 7, 300, 64], new, holes=[(0, 3), (1, 16)])
    paged(dev, p, window=window, sinks=sinks, weights=rng.random((5, kv_heads, p.cap), dtype=np.float32))
