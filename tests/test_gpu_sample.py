"""Sampling against its definition in 64 bits.  Tokens are compared exactly: the kernel's weights are off by less than 2^-44 of themselves and 2^-47 of the largest, so
that a given uniform number falls on the other side of a border once in 10^7 rows or more; probabilities within that and the rounding to 32 bits."""
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


def choose(x, u, temperature, k, p, min_p):
    """one row in 64 bits: the token and its share"""
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return -1, 0.0
    if x.max() == np.inf:
        x = np.where(x == np.inf, 0.0, -np.inf)
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / temperature))
    order = np.argsort(-x, kind="stable")
    n = len(x)
    if 0 < k < n:
        n = k
    if p < 1:
        front = w[order[:n]]
        before = np.concatenate([[0.0], np.cumsum(front)[:-1]])
        n = max(1, int((before < p * front.sum()).sum()))
    if min_p > 0:
        n = min(n, int((w[order] >= min(min_p, 1.0)).sum()))
    kept = np.zeros_like(w)
    kept[order[:n]] = w[order[:n]]
    sums = np.cumsum(kept)
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    token = int(np.searchsorted(sums, u * sums[-1], side="right"))
    return token, kept[token] / sums[-1]


def run(dev, x, dtype, u, temperature=None, k=None, p=None, min_p=None, stride=None, shift=0):
    """x [rows, vocab], already of the type; the settings are numbers or arrays"""
    rows, vocab = x.shape
    stride = stride or vocab
    whole = np.full(shift + rows * stride, 100.0)               # what lies between the rows would win
    for r in range(rows):
        whole[shift + r * stride:shift + r * stride + vocab] = x[r]
    buf = ref.upload(dev, whole, dtype)
    row = lambda v, t: None if v is None else np.ascontiguousarray(np.broadcast_to(np.asarray(v, t), (rows,)))        # noqa: E731
    u, temperature, k, p, min_p = row(u, np.float32), row(temperature, np.float32), row(k, np.int32), row(p, np.float32), row(min_p, np.float32)
    on = [None if v is None else dev.upload(v) for v in (temperature, k, p, min_p)]
    probs = dev.empty((rows,), _lib.F32)
    got = dev.sample(buf.view(shift, (rows, vocab)), dev.upload(u), *on, row_stride=stride, probs=probs).to_numpy()
    probs = probs.to_numpy()
    for r in range(rows):
        at = lambda v, none: none if v is None else float(v[r])        # noqa: E731
        want, share = choose(x[r], float(u[r]), at(temperature, 1.0), int(at(k, 0)), at(p, 1.0), at(min_p, 0.0))
        assert got[r] == want, (r, got[r], want, float(u[r]), at(temperature, None), at(k, None), at(p, None), at(min_p, None))
        assert abs(probs[r] - share) <= 2.0 ** -23 * share + 1e-12, (r, probs[r], share)
    return got


def logits(rng, rows, vocab, dtype, peaks=True):
    x = rng.standard_normal((rows, vocab)) * 2.2 - 4
    if peaks:
        for r in range(rows):
            x[r, rng.integers(0, vocab, 8)] += rng.random() * 14
    return ref.rounded(x, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 100, 1000, 1025, 4099, 16384, 32064, 51865, 65536, 65537, 131071])
@pytest.mark.parametrize("settings", [dict(), dict(k=40), dict(p=0.9), dict(min_p=0.05), dict(k=50, p=0.95, min_p=0.02), dict(temperature=0.0), dict(k=1)])
def test_sizes(dev, dtype, vocab, settings):
    rng = np.random.default_rng(vocab)
    rows = 5
    x = logits(rng, rows, vocab, dtype)
    run(dev, x, dtype, rng.random(rows), **{"temperature": [0.3, 0.7, 1.0, 1.3, 3.0], **settings})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [2, 3, 63, 64, 65, 999, 1000, 1023, 1024, 1025, 5000, 19999, 20000, 20001, 2 ** 31 - 1, 0, -1, -2 ** 31])
def test_top_k(dev, dtype, k):
    rng = np.random.default_rng(k % 1000)
    run(dev, logits(rng, 6, 20000, dtype), dtype, rng.random(6), 1.5, k)
    run(dev, logits(rng, 6, 20000, dtype, False), dtype, rng.random(6), 5.0, k, 0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 2, 50, 511, 512, 513, 900])
def test_top_k_of_rows_in_an_order(dev, dtype, k):
    """falling, rising, all but some alike, all in one place, few that are finite, ends of the range"""
    rng = np.random.default_rng(k)
    n = 20000
    x = np.sort(rng.standard_normal((8, n)) * 3, axis=1)
    x[0] = x[0, ::-1]
    x[1] = x[1, ::-1] - np.log1p(np.arange(n))
    x[3] = 1.0
    x[3, ::37] = 2.0
    x[4, :] = -4.0
    x[4, 7000:7600] = rng.standard_normal(600)
    x[5, :] = -np.inf
    x[5, rng.integers(0, n, 300)] = rng.standard_normal(300)
    x[6, ::2] = -6e4 if dtype == "f16" else -3.3e38
    x[6, 1::5] = 6e4 if dtype == "f16" else 3.3e38
    x[7] = 1.0
    x = ref.rounded(x, dtype)
    for p in (1.0, 0.9):
        run(dev, x, dtype, rng.random(8), k=k, p=p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [0.0, -1.0, 1e-30, 1e-6, 0.1, 0.5, 0.9, 0.999, 1 - 2.0 ** -24, 1.0, 1.5, np.nan])
def test_top_p(dev, dtype, p):
    rng = np.random.default_rng(7)
    x = logits(rng, 8, 12000, dtype)
    run(dev, x, dtype, rng.random(8), [0.05, 0.5, 1, 1, 2, 10, 1000, 1e6], None, p)
    run(dev, x, dtype, rng.random(8), [0.05, 0.5, 1, 1, 2, 10, 1000, 1e6], 300, p)


@pytest.mark.parametrize("dtype", DTYPES)
def test_each_row_its_own(dev, dtype):
    rng = np.random.default_rng(8)
    rows = 64
    x = logits(rng, rows, 5003, dtype)
    run(dev, x, dtype, rng.random(rows), np.where(rng.random(rows) < 0.2, 0.0, rng.random(rows) * 2), rng.integers(-2, 200, rows), rng.random(rows) * 1.2, rng.random(rows) * 0.1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("values", [1, 2, 5, 40])
@pytest.mark.parametrize("vocab", [50, 3000, 40000])
def test_ties(dev, dtype, values, vocab):
    """rows of a few values: cuts and choices lie among equals, and the lower index goes first"""
    rng = np.random.default_rng(values)
    x = ref.rounded(rng.integers(0, values, (6, vocab)) * 0.5, dtype)
    u = [0.0, 0.25, 0.5, 0.75, 0.999, 1 - 2.0 ** -24]
    run(dev, x, dtype, u)
    run(dev, x, dtype, u, 1.0, [1, 2, vocab // 3, vocab // 2 + 1, vocab - 1, 7])
    run(dev, x, dtype, u, 0.5, None, [0.25, 0.5, 0.75, 0.9, 0.01, 0.999])
    run(dev, x, dtype, u, 2.0, [vocab // 2 + 1] * 6, [0.25, 0.5, 0.75, 0.9, 0.01, 0.999], 0.5)
    run(dev, x, dtype, u, 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_finite(dev, dtype):
    rng = np.random.default_rng(9)
    x = logits(rng, 12, 3001, dtype)
    lowest = {"f32": -3.4e38, "f16": -65504.0, "bf16": -3.38e38}[dtype]
    x[0] = -np.inf                                              # nothing to choose from
    x[1] = np.nan
    x[2, ::2], x[2, 1::2] = np.nan, -np.inf
    x[3, rng.integers(0, 3001, 2900)] = -np.inf
    x[4, rng.integers(0, 3001, 2900)] = np.nan
    x[5, 10:], x[5, 3] = -np.inf, np.nan
    x[6, [7, 100, 2000]] = np.inf                               # they share the weight
    x[7, 3000], x[7, :3000] = np.inf, np.nan
    x[8, 5:] = lowest
    x[9] = lowest
    x[10, rng.integers(0, 3001, 2000)] = lowest
    x[11] = -x[11] * 1000
    x = ref.rounded(x, dtype)
    u = rng.random(12)
    for settings in (dict(), dict(k=50), dict(k=2000), dict(p=0.8), dict(k=20, p=0.8, min_p=0.1), dict(min_p=0.5), dict(temperature=0.0), dict(temperature=np.inf), dict(temperature=1e-40),
                     dict(temperature=np.nan), dict(temperature=-1.0), dict(temperature=np.inf, p=0.5, k=100), dict(temperature=1e-40, p=0.5, k=3), dict(k=1500, p=0.5)):
        run(dev, x, dtype, u, **settings)


@pytest.mark.parametrize("dtype", DTYPES)
def test_uniform_numbers_at_the_ends(dev, dtype):
    rng = np.random.default_rng(10)
    x = logits(rng, 8, 999, dtype, False)
    u = [0.0, -0.0, -1.0, 1.0, 2.0, np.nan, 1 - 2.0 ** -24, 1e-45]
    run(dev, x, dtype, u)
    run(dev, x, dtype, u, 1.0, 10)
    x[:, 0] = x[:, -1] = -np.inf
    run(dev, x, dtype, u, 1.0, None, 0.9)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("min_p", [0.0, -1.0, 1e-30, 0.01, 0.5, 1.0, 2.0, np.nan])
def test_min_p(dev, dtype, min_p):
    rng = np.random.default_rng(11)
    run(dev, logits(rng, 8, 4000, dtype), dtype, rng.random(8), [0.1, 0.5, 1, 2, 5, 100, 1, 1], None, None, min_p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stride, shift", [(3000, 0), (3001, 0), (3007, 1), (3500, 3), (3008, 5), (4000, 7)])
def test_strides_and_offsets(dev, dtype, stride, shift):
    rng = np.random.default_rng(stride)
    x = logits(rng, 5, 3000, dtype)
    run(dev, x, dtype, rng.random(5), 1.0, stride=stride, shift=shift)
    run(dev, x, dtype, rng.random(5), 1.0, 30, 0.9, stride=stride, shift=shift)


def test_rows_over_each_other(dev):
    """a stride of 0: one row of logits, many tokens of it"""
    rng = np.random.default_rng(12)
    x = logits(rng, 1, 5000, "f32")
    u = rng.random(300).astype(np.float32)
    got = dev.sample(dev.upload(x.astype(np.float32)).view(0, (1, 5000)), dev.upload(u[:1]))
    buf = dev.upload(np.tile(x.astype(np.float32), (300, 1)))
    many = dev.empty((300,), _lib.I32)
    _lib.check(dev.lib.rt_sample(dev.handle, _lib.F32, buf.ptr, 0, 300, 5000, None, None, None, None, dev.upload(u).ptr, many.ptr, None))
    want = [choose(x[0], float(v), 1.0, 0, 1.0, 0.0)[0] for v in u]
    assert many.to_numpy().tolist() == want and got.to_numpy()[0] == want[0]


def test_shares_of_many_draws(dev):
    """the frequencies of evenly spread numbers are the weights' shares"""
    x = np.array([[0.0, 1.0, -np.inf, 3.0, 2.0]], np.float32)
    n = 4096
    got = dev.sample(dev.upload(np.repeat(x, n, 0)), dev.upload(((np.arange(n) + 0.5) / n).astype(np.float32))).to_numpy()
    share = np.exp(x[0]) / np.exp(x[0]).sum()
    assert (np.abs(np.bincount(got, minlength=5) / n - share) <= 1.0 / n).all() and (np.diff(got) >= 0).all()


def test_recorded(dev):
    rng = np.random.default_rng(13)
    x, u = dev.upload(logits(rng, 9, 4000, "f32").astype(np.float32)), dev.upload(rng.random(9).astype(np.float32))
    k, p, out = dev.upload(np.full(9, 30, np.int32)), dev.upload(np.full(9, 0.9, np.float32)), dev.empty((9,), _lib.I32)
    with dev.capture() as graph:
        dev.sample(x, u, None, k, p, out=out)
    for _ in range(4):
        u.reshape((9,)).upload(rng.random(9).astype(np.float32))
        k.reshape((9,)).upload(rng.integers(0, 100, 9).astype(np.int32))
        graph.launch()
        got = out.to_numpy()
        assert np.array_equal(dev.sample(x, u, None, k, p).to_numpy(), got)


@pytest.mark.parametrize("dtype, vocab", [("f32", 1000003), ("f16", 1 << 24), ("bf16", 3000001)])
def test_large_vocabularies(dev, dtype, vocab):
    rng = np.random.default_rng(14)
    x = ref.rounded(rng.standard_normal((2, vocab)) * 3, dtype)
    u = rng.random(2)
    for settings in (dict(), dict(k=100), dict(p=0.5), dict(k=20000, p=0.9, min_p=1e-4), dict(temperature=0.0)):
        run(dev, x, dtype, u, **settings)


@pytest.mark.parametrize("dtype", DTYPES)
def test_twice_is_the_same(dev, dtype):
    """lists fill in any order, and sums add up in any: the bits of tokens and shares do not change"""
    rng = np.random.default_rng(15)
    x, u = ref.upload(dev, logits(rng, 64, 30011, dtype), dtype), dev.upload(rng.random(64).astype(np.float32))
    p, k = dev.upload(np.full(64, 0.95, np.float32)), dev.upload(rng.integers(1, 3000, 64).astype(np.int32))
    for settings in (dict(), dict(top_p=p), dict(top_k=k), dict(top_k=k, top_p=p)):
        probs = dev.empty((64,), _lib.F32)
        first = dev.sample(x, u, probs=probs, **settings).to_numpy(), probs.to_numpy()
        for _ in range(5):
            again = dev.sample(x, u, probs=probs, **settings).to_numpy(), probs.to_numpy()
            assert np.array_equal(again[0], first[0]) and np.array_equal(again[1], first[1])
