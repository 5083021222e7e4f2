"""The paged cache's append and eviction: values are moved, so everything is compared bit for bit, and what a call may not touch as well."""
import numpy as np
import pytest

import attention_ref as ref
from ratchet_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ratchet_amd import Device

    d = Device(0)
    yield d
    d.close()


def host_append(p, k, v):
    for b in range(len(p.lens)):
        lo, hi = p.starts[b], p.starts[b + 1]
        for j in range(lo, hi):
            t = max(int(p.lens[b]), 0) - int(hi - j)
            if 0 <= t < p.cap and 0 <= p.table[b, t // p.page] < p.pages:
                page = p.table[b, t // p.page]
                p.k[page, :, t % p.page], p.v[page, :, t % p.page] = k[j], v[j]


def host_evict(p, weights, keep, first, recent, table_out=None):
    """changes p's pages and lens, returns the weights"""
    table_out = p.table if table_out is None else table_out
    out, k0, v0 = weights.copy(), p.k.copy(), p.v.copy()
    for b in range(len(p.lens)):
        n = int(np.clip(p.lens[b], 0, p.cap))
        for g in range(p.kv_heads):
            stay = ref.evicted(weights[b, g], n, keep, first, recent)
            out[b, g, :len(stay)] = weights[b, g, stay]
            for i, t in enumerate(stay):
                src, dst = p.table[b, t // p.page], table_out[b, i // p.page]
                if 0 <= dst < p.pages:
                    have = 0 <= src < p.pages
                    p.k[dst, g, i % p.page] = k0[src, g, t % p.page] if have else 0.0
                    p.v[dst, g, i % p.page] = v0[src, g, t % p.page] if have else 0.0
        p.lens[b] = min(n, keep)
    return out


def on_device(dev, p):
    return dev.paged_cache(ref.upload(dev, p.k, p.dtype), ref.upload(dev, p.v, p.dtype), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))


def same(buf, want, dtype):
    return np.array_equal(ref.values(buf.to_numpy(), dtype), want, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads, dim", [(2, 64), (3, 20), (1, 1), (8, 128), (2, 6), (5, 7)])
@pytest.mark.parametrize("page", [1, 16, 7])
def test_append(dev, dtype, heads, dim, page):
    rng = np.random.default_rng(dim + page)
    # a first token, a prompt, a later piece, nothing, a page that is missing, more new tokens than lens counts, tokens beyond the table
    p = ref.Paged(rng, dtype, heads, heads, dim, page, [1, 50, 40, 20, 40, 2, 33], [1, 50, 7, 0, 5, 4, 2], holes=[(4, 38 // page)], spare=0)
    p.lens[1] = p.cap + 3
    k, v = (ref.rounded(rng.standard_normal((p.tokens, heads, dim)), dtype) for _ in range(2))
    cache = on_device(dev, p)
    dev.paged_append(cache, dev.upload(p.starts), ref.upload(dev, k, dtype), ref.upload(dev, v, dtype))
    host_append(p, k, v)
    assert same(cache.k_pages, p.k, dtype) and same(cache.v_pages, p.v, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_append_from_a_projection(dev, dtype, pad):
    """k and v side by side with queries in rows of any pitch, rows of no sequence among them"""
    rng = np.random.default_rng(pad)
    p = ref.Paged(rng, dtype, 2, 2, 64, 16, [100, 9], [30, 1])
    p.starts = p.starts + 2
    rows = ref.rounded(rng.standard_normal((36, 6 * 64 + pad)), dtype)
    buf, strides = ref.upload(dev, rows, dtype), (6 * 64 + pad, 64)
    cache = on_device(dev, p)
    dev.paged_append(cache, dev.upload(p.starts), buf.view(128, (36, 2, 64)), buf.view(256, (36, 2, 64)), k_strides=strides, v_strides=strides)
    host_append(p, rows[:, 128:256].reshape(36, 2, 64), rows[:, 256:384].reshape(36, 2, 64))
    assert same(cache.k_pages, p.k, dtype) and same(cache.v_pages, p.v, dtype)


@pytest.mark.parametrize("seqs", [64, 65, 5000])
def test_append_to_many_sequences(dev, seqs):
    rng = np.random.default_rng(seqs)
    lens = rng.integers(1, 30, seqs)
    p = ref.Paged(rng, "f16", 1, 1, 8, 8, lens, np.minimum(rng.integers(0, 3, seqs), lens))
    k, v = (ref.rounded(rng.standard_normal((p.tokens, 1, 8)), "f16") for _ in range(2))
    cache = on_device(dev, p)
    dev.paged_append(cache, dev.upload(p.starts), ref.upload(dev, k, "f16"), ref.upload(dev, v, "f16"))
    host_append(p, k, v)
    assert same(cache.k_pages, p.k, "f16") and same(cache.v_pages, p.v, "f16")


def weights_of(rng, shape, kind):
    w = rng.random(shape, dtype=np.float32)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "few":
        w = np.round(w * 4).astype(np.float32) / 4
    elif kind == "odd":                                         # zeros of both signs, negative values, infinities, NaN
        w = np.where(w < 0.2, np.float32(-0.0), np.where(w < 0.4, np.float32(0.0), w - 0.7)).astype(np.float32)
        w[..., 5::17], w[..., 6::23], w[..., 7::29] = np.nan, np.inf, -np.inf
    elif kind == "near":                                        # values that differ in their last bits
        w = (np.float32(1.0).view(np.uint32) + rng.integers(0, 600, shape).astype(np.uint32)).view(np.float32)
    return w


@pytest.mark.parametrize("dtype, dim", [("f16", 64), ("bf16", 80), ("f32", 20), ("f16", 7)])
@pytest.mark.parametrize("kind", ["any", "equal", "few", "odd", "near"])
@pytest.mark.parametrize("where", ["in place", "elsewhere", "rows elsewhere"])
def test_evict(dev, dtype, dim, kind, where):
    rng = np.random.default_rng(dim)
    lens = [1500, 300, 40, 1, 0, 39, 41, 1100]
    p = ref.Paged(rng, dtype, 2, 2, dim, 16, lens, [1] * 8, extra_pages=40, holes=[(1, 2), (7, 5)])
    keep, first, recent = 40, 3, 9
    w = weights_of(rng, (8, 2, p.cap), kind)
    cache, w_dev = on_device(dev, p), dev.upload(w)
    if where == "in place":
        after = dev.paged_evict(cache, w_dev, keep, first, recent)
        assert after is cache
        want, w_out = host_evict(p, w, keep, first, recent), w_dev
    else:
        table = np.full(p.table.shape, -1, np.int32)
        for b in range(8):
            table[b, :3] = p.free[3 * b:3 * b + 3]
        table[3, 0], table[6, 1] = p.pages, -7                  # rows that go nowhere
        extra = {} if where == "rows elsewhere" else {"lens_out": dev.upload(np.full(8, -1, np.int32)), "weights_out": dev.upload(w)}
        after = dev.paged_evict(cache, w_dev, keep, first, recent, to=dev.upload(table), **extra)
        want, w_out = host_evict(p, w, keep, first, recent, table), extra.get("weights_out", w_dev)
        if extra:
            assert np.array_equal(w_dev.to_numpy().view(np.uint32), w.view(np.uint32)) and np.array_equal(cache.lens.to_numpy(), lens)
    assert np.array_equal(after.lens.to_numpy(), p.lens)
    assert np.array_equal(w_out.to_numpy().view(np.uint32), want.view(np.uint32))
    assert same(cache.k_pages, p.k, dtype) and same(cache.v_pages, p.v, dtype)


@pytest.mark.parametrize("keep, first, recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 64, 0), (64, 0, 64), (64, 30, 34), (1023, 0, 0), (1024, 4, 100), (2999, 1, 1), (3000, 0, 0)])
@pytest.mark.parametrize("kind", ["any", "few"])
def test_what_stays(dev, keep, first, recent, kind):
    rng = np.random.default_rng(keep)
    p = ref.Paged(rng, "f16", 1, 1, 8, 32, [3000, 2048, 65], [1, 1, 1])
    w = weights_of(rng, (3, 1, p.cap), kind)
    cache, w_dev = on_device(dev, p), dev.upload(w)
    dev.paged_evict(cache, w_dev, keep, first, recent)
    want = host_evict(p, w, keep, first, recent)
    assert np.array_equal(cache.lens.to_numpy(), p.lens) and np.array_equal(w_dev.to_numpy(), want)
    assert same(cache.k_pages, p.k, "f16") and same(cache.v_pages, p.v, "f16")


def test_evict_token_by_token(dev):
    """a cache held at its size: one token out for one token in, twenty times, recorded once"""
    rng = np.random.default_rng(2)
    p = ref.Paged(rng, "f16", 2, 2, 64, 16, [200, 150], [1, 1])
    w = rng.random((2, 2, p.cap), dtype=np.float32)
    cache, w_dev = on_device(dev, p), dev.upload(w)
    dev.paged_evict(cache, w_dev, 150, 2, 10)                   # eager once: the workspace is there
    w = host_evict(p, w, 150, 2, 10)
    with dev.capture() as graph:
        dev.paged_evict(cache, w_dev, 140, 2, 10)
    for step in range(4):
        p.lens = p.lens + 7
        now = p.lens.astype(np.int32)
        dev.lib.rt_h2d(dev.handle, cache.lens.ptr, now.ctypes.data, now.nbytes)
        graph.launch()
        w = host_evict(p, w, 140, 2, 10)
        assert np.array_equal(cache.lens.to_numpy(), p.lens) and np.array_equal(w_dev.to_numpy(), w), step
        assert same(cache.k_pages, p.k, "f16") and same(cache.v_pages, p.v, "f16"), step
        dev.sync()


@pytest.mark.parametrize("length", [100000])
def test_evict_a_long_sequence(dev, length):
    rng = np.random.default_rng(9)
    p = ref.Paged(rng, "f16", 1, 1, 8, 64, [length], [1])
    w = weights_of(rng, (1, 1, p.cap), "few")
    cache, w_dev = on_device(dev, p), dev.upload(w)
    dev.paged_evict(cache, w_dev, 30000, 4, 1000)
    want = host_evict(p, w, 30000, 4, 1000)
    assert np.array_equal(cache.lens.to_numpy(), p.lens) and np.array_equal(w_dev.to_numpy(), want)
    assert same(cache.k_pages, p.k, "f16") and same(cache.v_pages, p.v, "f16")
