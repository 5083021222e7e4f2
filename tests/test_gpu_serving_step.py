"""The operators of a generated token one after the other, as a server runs them: embedding row, rotary positions and append, capped attention over the pages, sampling; a prompt first,
then steps, eager and replayed from one graph.  Each step is checked from what the one before left on the device; the bounds are those of each operator's own tests."""
import numpy as np
import pytest

import attention_ref as ref
from ratchet_amd import _lib
from test_gpu_attention_scored import head, visible
from test_gpu_rope_tokens import turned
from test_gpu_sample import choose

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, ROTARY, PAGE, VOCAB, CAP = 8, 2, 64, 48, 16, 500, 12.0


class Server:
    """a cache for three sequences, an embedding that holds q, k and v of each token, and a last product"""

    def __init__(self, dev, dtype, seed):
        rng = np.random.default_rng(seed)
        self.dev, self.dtype, self.rng = dev, dtype, rng
        self.width = (HEADS + 2 * KV) * DIM
        self.embedding = ref.rounded(rng.standard_normal((VOCAB, self.width)), dtype)
        self.product = rng.standard_normal((HEADS * DIM, VOCAB)) * 0.2
        self.slopes = np.float32(2.0 ** (-np.arange(1, HEADS + 1)))
        self.prefix = np.array([0, 7, 20], np.int32)
        self.lens = np.zeros(3, np.int32)
        self.table_host = rng.permutation(24).astype(np.int32).reshape(3, 8)
        zeros = np.zeros((24, KV, PAGE, DIM))
        self.lens_dev = dev.upload(self.lens)
        self.cache = dev.paged_cache(ref.upload(dev, zeros, dtype), ref.upload(dev, zeros, dtype), dev.upload(self.table_host), self.lens_dev)
        self.on = {"embedding": ref.upload(dev, self.embedding, dtype), "slopes": dev.upload(self.slopes), "prefix": dev.upload(self.prefix), "turns": dev.rope_table(ROTARY, 10000.0, 4.0)}

    def embed(self, tokens_dev, n, qkv=None):
        """qkv rows of the tokens, gathered by index, and rotated, appended and attended to"""
        dev = self.dev
        qkv = dev.index_select(self.on["embedding"], tokens_dev, 0, out=qkv)
        q, k, v = (qkv.view(o * DIM, (n, h, DIM)) for o, h in ((0, HEADS), (HEADS, KV), (HEADS + KV, KV)))
        return qkv, q, k, v

    def step(self, tokens_dev, starts_dev, n, buffers=None):
        dev, s = self.dev, (self.width, DIM)
        b = buffers or {}
        qkv, q, k, v = self.embed(tokens_dev, n, b.get("qkv"))
        turned_q = dev.paged_rope_append(self.cache, starts_dev, q, k, v, self.on["turns"], factor=1.1, interleaved=True, q_strides=s, k_strides=s, v_strides=s, out=b.get("turned"))
        out = dev.paged_attention(turned_q, self.cache, starts_dev, out=b.get("out"), lse=b.get("lse"), cap=CAP, slopes=self.on["slopes"], prefix=self.on["prefix"])
        return qkv, turned_q, out

    def check(self, tokens, starts, turned_q, out):
        """queries, pages and the attention's results of a step, on the host"""
        d, rows = self.dtype, self.embedding[tokens].reshape(len(tokens), HEADS + 2 * KV, DIM)
        at = np.concatenate([self.lens[b] - (starts[b + 1] - starts[b]) + np.arange(starts[b + 1] - starts[b]) for b in range(3)])
        factor = float(np.float32(1.1))
        want, off = turned(rows[:, :HEADS + KV], at, ROTARY, 10000.0, np.full(ROTARY // 2, 4.0), factor, True, d)
        q = ref.values(turned_q.to_numpy(), d)
        ref.check(q, want[:, :HEADS], off[:, :HEADS], "q")
        k_pages, v_pages, o = (ref.values(x.to_numpy(), d) for x in (self.cache.k_pages, self.cache.v_pages, out))
        for b in range(3):
            t = np.arange(self.lens[b])
            k, v = (pages[self.table_host[b, t // PAGE], :, t % PAGE].transpose(1, 0, 2) for pages in (k_pages, v_pages))
            lo, hi = starts[b], starts[b + 1]
            new = slice(self.lens[b] - (hi - lo), self.lens[b])
            ref.check(k[:, new].transpose(1, 0, 2), want[lo:hi, HEADS:], off[lo:hi, HEADS:], "k")
            assert np.array_equal(v[:, new].transpose(1, 0, 2), rows[lo:hi, HEADS + KV:])
            shift = self.lens[b] - (hi - lo)
            see = visible(hi - lo, self.lens[b], shift, True, 0, 0, None, int(self.prefix[b]))
            distance = (np.arange(hi - lo) + shift)[:, None] - t[None, :]
            for h in range(HEADS):
                want_o, _, o_off, _ = head(q[lo:hi, h], k[h // (HEADS // KV)], v[h // (HEADS // KV)], see, DIM ** -0.5, d, CAP, float(self.slopes[h]), distance)
                ref.check(o[lo:hi, h], want_o, o_off, ("o", b, h))
        return o


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_prompts_and_steps(dtype):
    from ratchet_amd import Device

    dev = Device(0)
    s = Server(dev, dtype, 3)
    # three prompts, one of a single token, then steps of one token each
    new = np.array([30, 1, 77])
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tokens = s.rng.integers(0, VOCAB, starts[-1]).astype(np.int32)
    s.lens += new.astype(np.int32)
    s.lens_dev.reshape((3,)).upload(s.lens)
    _, q, out = s.step(dev.upload(tokens), dev.upload(starts), len(tokens))
    o = s.check(tokens, starts, q, out)[starts[1:] - 1]

    one = np.arange(4, dtype=np.int32)
    starts_dev, tokens_dev = dev.upload(one), dev.empty((3,), _lib.I32)
    logits_dev, uniform_dev = dev.upload(np.zeros((3, VOCAB), np.float32)), dev.upload(np.zeros(3, np.float32))
    settings = {"temperature": np.array([1.0, 0.0, 0.7], np.float32), "top_k": np.array([0, 5, 40], np.int32), "top_p": np.array([0.9, 1.0, 0.95], np.float32)}
    on = {k: dev.upload(v) for k, v in settings.items()}
    e = {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}[dtype]
    buffers = {"qkv": dev.empty((3, s.width), e), "turned": dev.empty((3, HEADS, DIM), e), "out": dev.empty((3, HEADS, DIM), e), "lse": dev.empty((3, HEADS), _lib.F32)}

    def run():
        dev.sample(logits_dev, uniform_dev, out=tokens_dev, **on)
        return s.step(tokens_dev, starts_dev, 3, buffers)

    run()                                                       # before it is recorded: workspaces are there
    with dev.capture() as graph:
        run()
    for number in range(12):
        logits = (o.reshape(3, -1) @ s.product).astype(np.float32)
        uniform = s.rng.random(3).astype(np.float32)
        logits_dev.reshape((3, VOCAB)).upload(logits)
        uniform_dev.reshape((3,)).upload(uniform)
        s.lens += 1
        s.lens_dev.reshape((3,)).upload(s.lens)
        if number % 3 == 2:
            run()
        else:
            graph.launch()
        got = tokens_dev.to_numpy()
        for r in range(3):
            assert got[r] == choose(logits[r].astype(np.float64), float(uniform[r]), float(settings["temperature"][r]), int(settings["top_k"][r]), float(settings["top_p"][r]), 0.0)[0]
        o = s.check(got, one, buffers["turned"], buffers["out"])
    dev.close()


def test_two_devices_at_once():
    """two devices of one GPU, each with its own stream and workspace, their calls interleaved"""
    from ratchet_amd import Device

    devs = [Device(0), Device(0)]
    rng = np.random.default_rng(4)
    q, k, v = (rng.standard_normal(n).astype(np.float16) for n in ((2, 8, 1, 128), (2, 2, 4000, 128), (2, 2, 4000, 128)))
    x, u = rng.standard_normal((16, 30000)).astype(np.float32), rng.random(16).astype(np.float32)
    rows, at = rng.standard_normal((500, 4, 64)).astype(np.float32), rng.integers(0, 10000, 500).astype(np.int32)
    held = []
    for d in devs:
        held.append({"qkv": [d.upload(a) for a in (q, k, v)], "logits": d.upload(x), "u": d.upload(u), "p": d.upload(np.full(16, 0.9, np.float32)), "rows": d.upload(rows), "at": d.upload(at),
                     "table": d.rope_table(64)})
    results = [[], []]
    for _ in range(20):
        for n, d in enumerate(devs):
            h = held[n]
            results[n].append((d.attention(*h["qkv"], cap=8.0), d.sample(h["logits"], h["u"], top_p=h["p"]), d.rope_tokens(h["rows"], h["at"], h["table"])))
    first = [r.to_numpy() for r in results[0][0]]
    for n in range(2):
        for r in results[n]:
            assert all(np.array_equal(a.to_numpy(), b) for a, b in zip(r, first))
    results.clear()
    held.clear()
    for d in devs:
        d.close()


def test_beyond_four_gibibytes():
    """offsets that pass 32 bits: rows of logits far apart, rows to rotate far apart, and keys of a long text"""
    from ratchet_amd import Device

    dev = Device(0)
    rng = np.random.default_rng(5)
    far = (1 << 31) + 24                                        # elements
    buf = dev.empty((2 * far + 5000,), _lib.F16)
    x = rng.standard_normal((3, 5000)).astype(np.float16)
    for r in range(3):
        buf.view(r * far, (5000,)).upload(x[r])
    u = rng.random(3).astype(np.float32)
    got = dev.sample(buf.view(0, (3, 5000)), dev.upload(u), row_stride=far).to_numpy()
    assert got.tolist() == [choose(x[r].astype(np.float64), float(u[r]), 1.0, 0, 1.0, 0.0)[0] for r in range(3)]
    rows, at = x[:, :4096].reshape(3, 32, 128).astype(np.float64), np.array([5, 70000, 3], np.int32)
    want, off = turned(rows, at, 128, 10000.0, None, 1.0, False, "f16")
    out = dev.rope_tokens(buf.view(0, (3, 32, 128)), dev.upload(at), dev.rope_table(128), strides=(far, 128), out=buf.view(0, (3, 32, 128)), out_strides=(far, 128))
    assert out is not None
    for r in range(3):
        ref.check(ref.values(buf.view(r * far, (32, 128)).to_numpy(), "f16"), want[r], off[r], ("rope", r))
    # 600 keys, the last of them 4 GiB behind the first
    step = (1 << 31) // 600 // 8 * 8 + 64
    k, v, q = (ref.rounded(rng.standard_normal(s), "f16") for s in ((1, 1, 600, 64), (1, 1, 600, 64), (1, 2, 5, 64)))
    for t in range(600):
        buf.view(t * step, (64,)).upload(k[0, 0, t].astype(np.float16))
        buf.view(far + t * step, (64,)).upload(v[0, 0, t].astype(np.float16))
    strides = (0, 0, step, 1)
    for queries in (q, q[:, :, :1]):
        n = queries.shape[2]
        got = dev.attention(ref.upload(dev, queries, "f16"), buf.view(0, k.shape), buf.view(far, v.shape), k_strides=strides, v_strides=strides, cap=6.0, documents=dev.upload(np.array([[0, 200, 600]], np.int32)))
        got = ref.values(got.to_numpy(), "f16")
        see = visible(n, 600, 600 - n, True, 0, 0, [0, 200, 600], None)
        for h in range(2):
            want, _, off, _ = head(queries[0, h], k[0, 0], v[0, 0], see, 0.125, "f16", 6.0)
            ref.check(got[0, h], want, off, ("o", h))
    dev.close()
