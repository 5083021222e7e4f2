"""Attention, append and eviction in 64 bits, and how far 32-bit sums and the element type's roundings can take a result from them.

Bounds, all worst cases.  u = 2^-24 is the half step of f32, e the half step of the element type (bf16 2^-8, f16 2^-11, f32 2^-24).
A score is a sum of D products, scaled: off by at most ds = c * (D + 4) * u * sum |q_d k_d|, with c = |scale|; the scale's own product, log2(e)
and the rounding of s - m add 4 u |s| each at most, in all ds <= c (D + 16) u sum |q_d k_d|.  A weight exp(s - m) / l is then off by a factor within
1 +- (2 ds_max + (n + 32) u): its own score and those in l, the n additions in l, exp2, the divide, and the rescaling of running sums by
tiles.  It is rounded to the element type once (e), the sum over the keys adds n roundings of u, the result rounds once more (e):
    |o - exact| <= e |o| + (e + 2 ds_max + (2 n + 64) u) sum w |v|        (+ the smallest subnormal's half step)
f16 weights below 2^-14 of the row's largest are subnormal: off by 2^-25 of the largest at most, which l >= 1 divides: + 2^-25 sum |v|.
    |lse - exact| <= ds_max + (n + 32) u + 4 u |lse|
    |received - exact| <= sum over its queries of w (2 ds_max + (n + 64) u + 8 u |lse|) + (queries + 1) u (sum w + old)"""
import numpy as np
import torch

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rounded(x, dtype):
    """float64 numpy array -> the nearest values of `dtype`, in float64"""
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(TORCH[dtype]).double().numpy()


def raw(x, dtype):
    """values of `dtype` as the array that Device.upload takes (bf16: its bits)"""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float64)).to(torch.float32).to(TORCH[dtype])
    return t.view(torch.int16).numpy().view(np.uint16) if dtype == "bf16" else t.numpy()


def upload(dev, x, dtype):
    return dev.upload(raw(x, dtype), bf16=dtype == "bf16")


def values(a, dtype):
    """what a download holds, in float64"""
    if dtype == "bf16":
        return (np.asarray(a).view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(a).astype(np.float64)


def visible(n, keys, shift, causal, window, sinks, holes=None):
    """[n, keys]: query j sits at position j + shift"""
    p, t = np.arange(n)[:, None] + shift, np.arange(keys)[None, :]
    see = np.broadcast_to(t <= p, (n, keys)) if causal else np.ones((n, keys), bool)
    if window:
        see = see & ((p - t < window) | (t < sinks))
    return see & ~holes[None, :] if holes is not None else see


def head(q, k, v, see, scale, dtype):
    """one head: o, lse, the weights, and the bounds of o and of each row's lse, and of a weight's factor"""
    n, d = q.shape
    keys = k.shape[0]
    o, lse, w = np.zeros((n, v.shape[1])), np.full(n, -np.inf), np.zeros((n, keys))
    o_off, lse_off, factor = np.zeros_like(o), np.zeros(n), np.zeros(n)
    some = see.any(axis=1) if keys else np.zeros(n, bool)
    if some.any():
        with np.errstate(invalid="ignore"):
            s = np.where(see, (q @ k.T) * scale, -np.inf)
            mass = np.where(see, np.abs(q) @ np.abs(k).T, 0.0).max(axis=1) * abs(scale) * (d + 16) * U
        m = np.where(some, s.max(axis=1), 0.0)
        x = np.exp(s - m[:, None])
        total = x.sum(axis=1)
        w = x / np.where(some, total, 1.0)[:, None]
        lse = np.where(some, np.log(np.where(some, total, 1.0)) + m, -np.inf)
        v0 = np.where(see.any(axis=0)[:, None], v, 0.0)
        o = w @ v0
        e = HALF_STEP[dtype]
        seen = see.sum(axis=1)
        o_off = e * np.abs(o) + (e + 2 * mass + (2 * seen + 64) * U)[:, None] * (w @ np.abs(v0)) + TINY[dtype]
        if dtype == "f16":
            o_off = o_off + 2.0 ** -25 * (see.astype(float) @ np.abs(v0))
        lse_off = mass + (seen + 32) * U + 4 * U * np.abs(np.where(some, lse, 0.0))
        factor = 2 * mass + (seen + 64) * U + 8 * U * np.abs(np.where(some, lse, 0.0))
    return o, lse, w, o_off, lse_off, factor


def check(got, want, off, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    exact = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, "NaN in other places", int((np.isnan(got) != np.isnan(want)).sum()))
    assert np.array_equal(got[exact & ~np.isnan(want)], want[exact & ~np.isnan(want)]), (what, "infinities differ")
    far = np.where(exact, 0.0, np.abs(np.where(exact, 0.0, got) - np.where(exact, 0.0, want)) - off)
    assert (far <= 0).all(), (what, "worst at", np.unravel_index(int(np.argmax(far)), far.shape), "by", float(far.max()), "bad", int((far > 0).sum()), "of", far.size)


class Paged:
    """A paged problem on the host: pages, tables, new tokens, and its answers."""

    def __init__(self, rng, dtype, heads, kv_heads, dim, page, lens, new, extra_pages=3, spare=1, spread=1.0, holes=()):
        self.dtype, self.heads, self.kv_heads, self.dim, self.page = dtype, heads, kv_heads, dim, page
        self.lens, self.new = np.asarray(lens), np.asarray(new)
        each = np.maximum(-(-self.lens // page), 0)
        self.table_len = int(each.max()) + spare
        self.pages = int(each.sum()) + extra_pages
        self.cap = self.table_len * page
        order = rng.permutation(self.pages)
        self.free = order[int(each.sum()):]
        self.table = np.full((len(self.lens), self.table_len), -1, np.int32)
        at = 0
        for b, n in enumerate(each):
            self.table[b, :n] = order[at:at + n]
            at += n
        for b, i in holes:
            self.table[b, i] = -1 if (b + i) % 2 else self.pages + 5
        shape = (self.pages, kv_heads, page, dim)
        self.k, self.v = rounded(rng.standard_normal(shape), dtype), rounded(rng.standard_normal(shape), dtype)
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.tokens = int(self.starts[-1])
        self.q = rounded(spread * rng.standard_normal((self.tokens, heads, dim)), dtype)

    def rows(self, pages, b):
        """[kv_heads, keys, dim] of sequence b and which of them have no page"""
        n = int(np.clip(self.lens[b], 0, self.cap))
        t = np.arange(n)
        page = self.table[b, t // self.page]
        gone = (page < 0) | (page >= self.pages)
        return np.where(gone[None, :, None], 0.0, pages[np.where(gone, 0, page), :, t % self.page].transpose(1, 0, 2)), gone

    def attention(self, scale, window=0, sinks=0, weights=None):
        """o, lse (with what is left as it was: NaN), received weights, and their bounds"""
        g = self.heads // self.kv_heads
        o, lse = np.full(self.q.shape, np.nan), np.full(self.q.shape[:2], np.nan)
        o_off, lse_off = np.zeros(o.shape), np.zeros(lse.shape)
        received = None if weights is None else weights.astype(np.float64).copy()
        r_off = None if weights is None else np.zeros(weights.shape)
        for b in range(len(self.lens)):
            lo, hi = self.starts[b], self.starts[b + 1]
            k, gone = self.rows(self.k, b)
            v, _ = self.rows(self.v, b)
            keys, shift = k.shape[1], int(max(self.lens[b], 0)) - int(hi - lo)
            see = visible(hi - lo, keys, shift, True, window, sinks, gone)
            if weights is not None:
                received[b, :, max(shift, 0):keys] = 0.0
            for h in range(self.heads):
                o[lo:hi, h], lse[lo:hi, h], w, o_off[lo:hi, h], lse_off[lo:hi, h], factor = head(self.q[lo:hi, h], k[h // g], v[h // g], see, scale, self.dtype)
                if weights is not None and keys:
                    received[b, h // g, :keys] += w.sum(axis=0)
                    r_off[b, h // g, :keys] += (w * factor[:, None]).sum(axis=0)
            if weights is not None and keys:
                r_off[b, :, :keys] += ((hi - lo) * g + 1) * U * np.abs(received[b, :, :keys])
        return o, lse, received, o_off, lse_off, r_off


def evicted(weights, length, keep, first, recent):
    """tokens of one KV head that stay"""
    if length <= keep:
        return np.arange(length)
    w = np.where(np.isnan(weights[:length]), -np.inf, weights[:length].astype(np.float64))
    nan_last = np.isnan(weights[:length])
    middle = np.arange(first, length - recent)
    order = sorted(middle, key=lambda t: (bool(nan_last[t]), -w[t], t))
    return np.array(sorted(list(range(first)) + list(order[:keep - first - recent]) + list(range(length - recent, length))), dtype=np.int64)
