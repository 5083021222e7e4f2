"""Calls of more rows than one grid of blocks has threads for (2^32 of a launch)."""
import numpy as np
import pytest

from ratchet_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ratchet_amd import Device

    d = Device(0)
    yield d
    d.close()


def test_append_of_more_than_2_to_the_24_tokens(dev):
    tokens, page = (1 << 24) + 77, 64
    rng = np.random.default_rng(0)
    pages = -(-tokens // page)
    order = rng.permutation(pages).astype(np.int32)
    rows = [rng.integers(0, 1 << 16, (tokens, 1, 1), dtype=np.uint16).view(np.float16) for _ in range(2)]
    k, v = (dev.empty((pages, 1, page, 1), _lib.F16).zero_() for _ in range(2))
    cache = dev.paged_cache(k, v, dev.upload(order[None]), dev.upload(np.array([tokens], np.int32)))
    dev.paged_append(cache, dev.upload(np.array([0, tokens], np.int32)), *(dev.upload(x) for x in rows))
    for buf, x in zip((k, v), rows):
        want = np.zeros(pages * page, np.uint16)
        want[:tokens] = x.view(np.uint16).ravel()
        got = buf.to_numpy().view(np.uint16).reshape(pages, page)
        assert np.array_equal(got[order], want.reshape(pages, page))


def test_attention_of_more_than_2_to_the_26_rows(dev):
    """one key, so that every row is that key's value"""
    rows = (1 << 26) + 5
    q = dev.empty((1, 1, rows, 1), _lib.F16).zero_()
    k, v = dev.upload(np.full((1, 1, 1, 1), 2.0, np.float16)), dev.upload(np.full((1, 1, 1, 1), 3.5, np.float16))
    out = dev.empty(q.shape, _lib.F16).zero_()
    dev.attention(q, k, v, causal=False, out=out)
    assert (out.to_numpy() == 3.5).all()


def test_attention_of_more_than_2_to_the_24_heads(dev):
    """of whole vectors of columns, each with one query and one key of its own"""
    shape = (65535, 257, 1, 8)
    rng = np.random.default_rng(1)
    x = rng.integers(0, 1000, shape, dtype=np.int16).astype(np.float16)
    v = dev.upload(x)
    assert np.array_equal(dev.attention(v, v, v).to_numpy(), x)
