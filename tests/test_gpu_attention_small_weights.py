"""f16 rows whose keys but one weigh less than f16's smallest number against the largest: together they are most of the result, as the key
they vanish against holds zeros."""
import numpy as np
import pytest

import attention_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ratchet_amd import Device

    d = Device(0)
    yield d
    d.close()


def rows(rng, queries, heads, keys, dim, far):
    """queries of one direction; key 0 lies `far` (in scores) above the others, its value is 0"""
    q, k = 0.1 * rng.standard_normal((queries, heads, dim)), 0.1 * rng.standard_normal((keys, heads, dim))
    v = 500.0 * (1.0 + rng.random((keys, heads, dim)))
    q[:, :, 0], k[:, :, 0], v[0] = 8.0, 0.05 * rng.standard_normal((keys, heads)), 0.0
    k[0, :, 0] = far
    return (ref.rounded(x, "f16") for x in (q, k, v))


def bound(off, see, v):
    """attention_ref's without the half step of f16 weights of up to 1.  They are held as multiples of 2^-24 of the row's largest running m
    times 2^6 at least, which is what the largest weight is: off by 2^-25 / 2^6 of it, 2^-31 sum |v| after the division"""
    total = see.astype(float) @ np.abs(v)
    return off - 2.0 ** -25 * total + 2.0 ** -31 * total


@pytest.mark.parametrize("far", [15.0, 17.5, 19.0])
@pytest.mark.parametrize("queries, keys", [(1, 3000), (1, 100), (200, 3000), (700, 900)])
def test_contiguous(dev, far, queries, keys):
    rng = np.random.default_rng(queries)
    q, k, v = rows(rng, queries, 2, keys, 64, far)
    got = ref.values(dev.attention(*(ref.upload(dev, x.transpose(1, 0, 2)[None], "f16") for x in (q, k, v)), scale=0.125).to_numpy(), "f16")
    see = ref.visible(queries, keys, keys - queries, True, 0, 0)
    for h in range(2):
        o, _, _, off, _, _ = ref.head(q[:, h], k[:, h], v[:, h], see, 0.125, "f16")
        ref.check(got[0, h], o, bound(off, see, v[:, h]), h)


@pytest.mark.parametrize("far", [17.5, 19.0])
@pytest.mark.parametrize("new", [1, 300])
def test_paged(dev, far, new):
    """shared out over blocks and joined"""
    rng = np.random.default_rng(new)
    p = ref.Paged(rng, "f16", 2, 2, 64, 16, [6000, 40], [new, 1])
    q, k, v = rows(rng, new, 2, 6000, 64, far)
    p.q[:new] = q
    t = np.arange(6000)
    p.k[p.table[0, t // 16], :, t % 16], p.v[p.table[0, t // 16], :, t % 16] = k, v
    cache = dev.paged_cache(ref.upload(dev, p.k, "f16"), ref.upload(dev, p.v, "f16"), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    got = ref.values(dev.paged_attention(ref.upload(dev, p.q, "f16"), cache, dev.upload(p.starts), scale=0.125).to_numpy(), "f16")
    see = ref.visible(new, 6000, 6000 - new, True, 0, 0)
    for h in range(2):
        o, _, _, off, _, _ = ref.head(q[:, h], k[:, h], v[:, h], see, 0.125, "f16")
        ref.check(got[:new, h], o, bound(off, see, v[:, h]), h)
