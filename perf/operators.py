"""Cases of the attention operators and of the paged KV cache they read: attention of encoders and prompts with a sliding window
and sinks, tokens and chunks over a paged cache, the append to it and the eviction from it by accumulated attention weight.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program has in hand before the call
and run() is one pass: the framework's call where `own` is true, the formulas in plain torch operations otherwise."""
import math

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MOST_SCORES = 2.2e9        # (query, key, head) triples of the largest listed case, padding included
MOST_BYTES = 2.2e9         # bytes of cache rows in the largest listed case

_open = {}


def _device():
    if "dev" not in _open:
        from ratchet_amd import Device
        _open["dev"] = Device(0)
    return _open["dev"]


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # attention of a Whisper-tiny encoder over four 30 s windows, f32, every frame sees every frame
        {"name": "encoder_f32", "kind": "attention", "dtype": "f32", "batch": 4, "heads": 6, "kv_heads": 6, "dim": 64, "queries": 1500, "keys": 1500,
         "causal": False, "window": 0, "sinks": 0},
        # a 2048-token Phi-2 prompt, q, k and v side by side as the projection leaves them
        {"name": "prompt_phi2_f16", "kind": "attention", "dtype": "f16", "batch": 1, "heads": 32, "kv_heads": 32, "dim": 80, "queries": 2048, "keys": 2048,
         "causal": True, "window": 0, "sinks": 0},
        # an 8192-token Phi-3 prompt with that model's sliding window of 2047 and four first tokens kept in sight: the largest case
        {"name": "prompt_window_phi3_bf16", "kind": "attention", "dtype": "bf16", "batch": 1, "heads": 32, "kv_heads": 32, "dim": 96, "queries": 8192,
         "keys": 8192, "causal": True, "window": 2047, "sinks": 4},
        # the next token of one long Phi-3 conversation, sliding window and sinks: latency of a generated token
        {"name": "token_window_phi3_f16", "kind": "paged", "dtype": "f16", "seqs": 1, "chunks": 0, "chunk": 0, "shortest": 7001, "longest": 7001, "heads": 32,
         "kv_heads": 32, "dim": 96, "page": 32, "window": 2047, "sinks": 4, "weights": False, "mix": 1},
        # one token for each of 64 conversations of 200 to 8000 tokens, four query heads to a KV head
        {"name": "tokens_64_bf16", "kind": "paged", "dtype": "bf16", "seqs": 64, "chunks": 0, "chunk": 0, "shortest": 200, "longest": 8000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "sinks": 0, "weights": False, "mix": 2},
        # a serving step: pieces of four prompts of up to 250 tokens next to twelve generated tokens
        {"name": "chunks_and_tokens_bf16", "kind": "paged", "dtype": "bf16", "seqs": 16, "chunks": 4, "chunk": 250, "shortest": 300, "longest": 8000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "sinks": 0, "weights": False, "mix": 3},
        # one token for each of 16 conversations whose keys are weighed for eviction
        {"name": "tokens_16_weights_bf16", "kind": "paged", "dtype": "bf16", "seqs": 16, "chunks": 0, "chunk": 0, "shortest": 500, "longest": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0, "weights": True, "mix": 4},
        # two Phi-2 prompts whose keys are weighed while they are read in
        {"name": "prompts_weights_phi2_f16", "kind": "paged", "dtype": "f16", "seqs": 2, "chunks": 2, "chunk": 1900, "shortest": 1, "longest": 1900, "heads": 32,
         "kv_heads": 32, "dim": 80, "page": 32, "window": 0, "sinks": 0, "weights": True, "mix": 5},
        # keys and values of the tokens of 64 conversations into the cache: the smallest call
        {"name": "append_tokens_64_bf16", "kind": "append", "dtype": "bf16", "seqs": 64, "chunks": 0, "chunk": 0, "shortest": 200, "longest": 2000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "mix": 6},
        # keys and values of four Phi-3 prompts of up to 2048 tokens into the cache
        {"name": "append_prompts_phi3_f16", "kind": "append", "dtype": "f16", "seqs": 4, "chunks": 4, "chunk": 2048, "shortest": 1, "longest": 2048, "heads": 32,
         "kv_heads": 32, "dim": 96, "page": 32, "mix": 7},
        # one long conversation cut to 1024 tokens
        {"name": "evict_1_bf16", "kind": "evict", "dtype": "bf16", "seqs": 1, "shortest": 4100, "longest": 4100, "kv_heads": 8, "dim": 128, "page": 16, "keep": 1024,
         "first": 4, "recent": 128, "mix": 8},
        # eight Phi-2 conversations of up to 4096 tokens cut to 2048 each
        {"name": "evict_8_phi2_f16", "kind": "evict", "dtype": "f16", "seqs": 8, "shortest": 1500, "longest": 4096, "kv_heads": 32, "dim": 80, "page": 32, "keep": 2048,
         "first": 4, "recent": 256, "mix": 9},
    ]


def _spread(rng, low, high):
    """log-uniform over [low, high]"""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    while True:
        kind = rng.choice(["attention", "attention", "paged", "paged", "paged", "append", "evict"])
        c = {"kind": kind, "dtype": rng.choice(["f16", "bf16", "f16", "bf16", "f32"])}
        heads, kv_heads = rng.choice([(6, 6), (8, 8), (32, 32), (32, 8), (16, 2), (12, 4)])
        dim, page, mix = rng.choice([64, 80, 96, 128, 40, 256]), rng.choice([16, 32, 64, 24, 128]), rng.randint(10, 10 ** 6)
        window = rng.choice([0, 0, _spread(rng, 16, 4096)])
        sinks = rng.choice([0, rng.randint(1, 64)]) if window else 0
        if kind == "attention":
            causal = rng.random() < 0.7
            queries = rng.choice([1, _spread(rng, 2, 6000)])
            c.update(batch=_spread(rng, 1, 8), heads=heads, kv_heads=kv_heads, dim=dim, queries=queries, keys=queries if rng.random() < 0.6 else _spread(rng, queries, 8000),
                     causal=causal, window=window if causal else 0, sinks=sinks if causal else 0)
        elif kind == "evict":
            longest = _spread(rng, 200, 8000)
            keep = _spread(rng, 64, longest)
            c.update(seqs=_spread(rng, 1, 16), shortest=rng.randint(1, longest), longest=longest, kv_heads=kv_heads, dim=dim, page=page, keep=keep, first=rng.choice([0, 4]),
                     recent=rng.randint(0, keep // 2), mix=mix)
        else:
            seqs, longest = _spread(rng, 1, 64), _spread(rng, 16, 8000)
            chunks = rng.choice([0, seqs, rng.randint(0, seqs)])
            c.update(seqs=seqs, chunks=chunks, chunk=_spread(rng, 2, 2048) if chunks else 0, shortest=rng.randint(1, longest), longest=longest, heads=heads, kv_heads=kv_heads,
                     dim=dim, page=page, mix=mix)
            if kind == "paged":
                c.update(window=window, sinks=sinks, weights=rng.random() < 0.3)
        if _fits(c):
            return c


def _fits(c):
    if c["kind"] == "attention":
        scores, rows = c["batch"] * c["heads"] * c["queries"] * c["keys"], c["batch"] * c["kv_heads"] * c["keys"]
    else:
        lens, new = _lengths(c)
        scores = len(lens) * c["heads"] * int(new.max()) * int(lens.max()) if c["kind"] == "paged" else 0
        rows = len(lens) * c["kv_heads"] * int(lens.max())
    return scores <= MOST_SCORES and 2 * rows * c["dim"] * BYTES[c["dtype"]] <= MOST_BYTES


def _lengths(c):
    """tokens in the cache of each sequence, the new ones among them, and how many are new"""
    r = np.random.RandomState(c["mix"])
    lens = r.randint(c["shortest"], c["longest"] + 1, c["seqs"])
    lens[r.randint(c["seqs"])] = c["longest"]
    new = np.ones_like(lens)
    if c.get("chunks"):
        at = r.permutation(c["seqs"])[:c["chunks"]]
        new[at] = r.randint(max(1, c["chunk"] // 2), c["chunk"] + 1, c["chunks"])
        new[at[0]] = c["chunk"]
        lens = np.maximum(lens, new)
    return lens, new


# ------------------------------------------------------------------------------------------------------------- prepare
class _Window:
    """What torch needs to see a device buffer of the library without a copy."""

    def __init__(self, buf, typestr):
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": buf.shape, "typestr": typestr, "data": (buf.ptr.value, False), "version": 2}


def _buffer(t):
    """`t` in a buffer of the library, and that buffer as torch sees it"""
    from ratchet_amd import _lib
    code, typestr = {torch.float32: (_lib.F32, "<f4"), torch.float16: (_lib.F16, "<f2"), torch.bfloat16: (_lib.BF16, "<i2"), torch.int32: (_lib.I32, "<i4")}[t.dtype]
    buf = _device().empty(tuple(t.shape), code)
    seen = torch.as_tensor(_Window(buf, typestr), device="cuda")
    seen = seen.view(torch.bfloat16) if t.dtype == torch.bfloat16 else seen
    seen.copy_(t)
    return buf, seen


def _inputs(c, seed):
    """the tensors of a case, made from the seed alone"""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, dtype = c["kind"], TORCH[c["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    def ints(v):
        return torch.as_tensor(np.ascontiguousarray(v, dtype=np.int32), device="cuda")

    if kind == "attention":
        b, h, g, d, n, k = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["queries"], c["keys"]
        t = {"q": normal(b, n, h, d) * 2, "k": normal(b, k, g, d), "v": normal(b, k, g, d)}
        if n == k:                                              # side by side, as one projection leaves them
            t = {"qkv": torch.cat([t["q"], t["k"], t["v"]], dim=2)}
        t["o"] = torch.zeros(b, n, h, d, device="cuda", dtype=dtype)
        return t
    lens, new = _lengths(c)
    g, d, page = c["kv_heads"], c["dim"], c["page"]
    each = -(-lens // page)                                     # pages of each sequence
    width = int(each.max()) + 2                                 # room in the table for what will be generated
    kept = -(-np.minimum(lens, c["keep"]) // page) if kind == "evict" else 0 * each
    total = int(each.sum() + kept.sum()) + 3
    order = np.random.RandomState(int(seed) % (1 << 31)).permutation(total)

    def table(count, first):
        out = np.full((len(lens), width), -1, np.int64)
        at = first + np.concatenate([[0], np.cumsum(count)])
        for i, n in enumerate(count):
            out[i, :n] = order[at[i]:at[i] + n]
        return ints(out)

    t = {"k_pages": normal(total, g, page, d), "v_pages": normal(total, g, page, d), "table": table(each, 0), "lens": ints(lens)}
    if kind == "evict":
        # sums of softmax rows: skewed, with many equal small values
        w = torch.rand(len(lens), g, width * page, generator=gen, device="cuda")
        t["weights"] = (w ** 8 * 4096).round() / 64
        t["to"], t["lens_out"], t["weights_out"] = table(kept, int(each.sum())), torch.zeros_like(t["lens"]), torch.zeros_like(t["weights"])
        return t
    t["starts"] = ints(np.concatenate([[0], np.cumsum(new)]))
    tokens = int(new.sum())
    t["qkv"] = torch.cat([normal(tokens, c["heads"], d) * 2, normal(tokens, 2 * g, d)], dim=1)
    if kind == "paged":
        t["o"] = torch.zeros(tokens, c["heads"], d, device="cuda", dtype=dtype)
        if c["weights"]:
            t["weights"] = torch.rand(len(lens), g, width * page, generator=gen, device="cuda")
            t["weights_out"] = torch.zeros_like(t["weights"])
    return t


def prepare(case, seed):
    c, t = case, _inputs(case, seed)
    s = {"case": c}
    if c["kind"] != "attention":
        lens, new = _lengths(c)
        s["longest"], s["most"] = int(lens.max()), int(new.max())
    if own:
        dev, both = _device(), {k: _buffer(v) for k, v in t.items()}
        b, s["seen"] = {k: v[0] for k, v in both.items()}, {k: v[1] for k, v in both.items()}
        d, g = c["dim"], c["kv_heads"]
        if c["kind"] == "attention":
            h, n, k = c["heads"], c["queries"], c["keys"]
            if "qkv" in b:
                w, at = h + 2 * g, (0, h * d, (h + g) * d)      # q, k and v are windows of the projection's rows
                s["q"], s["k"], s["v"] = (b["qkv"].view(o, (c["batch"], x, n, d)) for o, x in zip(at, (h, g, g)))
                s["q_strides"] = s["kv_strides"] = (n * w * d, d, w * d, 1)
            else:
                s["q"], s["k"], s["v"] = b["q"].reshape((c["batch"], h, n, d)), b["k"].reshape((c["batch"], g, k, d)), b["v"].reshape((c["batch"], g, k, d))
                s["q_strides"], s["kv_strides"] = (n * h * d, d, h * d, 1), (k * g * d, d, g * d, 1)
            s["o"], s["o_strides"] = b["o"].reshape((c["batch"], h, n, d)), (n * h * d, d, h * d, 1)
        else:
            s["cache"] = dev.paged_cache(b["k_pages"], b["v_pages"], b["table"], b["lens"])
            s.update({k: b.get(k) for k in ("starts", "o", "weights", "weights_out", "to", "lens_out")})
            if "qkv" in b:
                h, n = c["heads"], b["qkv"].shape[0]
                s["q"], s["k"], s["v"] = b["qkv"].view(0, (n, h, d)), b["qkv"].view(h * d, (n, g, d)), b["qkv"].view((h + g) * d, (n, g, d))
                s["strides"] = ((h + 2 * g) * d, d)
            if c["kind"] == "paged":
                s["lse"], s["seen"]["lse"] = _buffer(torch.zeros(n, h, device="cuda"))
    else:
        s["t"] = t
    return s


# ----------------------------------------------------------------------------------------------------------------- run
def run(state):
    c = state["case"]
    return {"attention": _attention, "paged": _paged, "append": _append, "evict": _evict}[c["kind"]](state, c)


def _heads_apart(t, c):
    """q, k and v as [batch, heads, tokens, dim] in 32 bits"""
    if "qkv" in t:
        q, k, v = t["qkv"].split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=2)
    else:
        q, k, v = t["q"], t["k"], t["v"]
    return [x.transpose(1, 2).float() for x in (q, k, v)]


def _weighted(q, k, v, visible, groups, scale):
    """softmax(scale q k^T) v where `visible`, in the inputs' type: q [b, heads, n, d], k and v [b, kv heads, t, d], visible [b or 1, n, t].
    Returns o [b, heads, n, d], lse [b, heads, n] and the weights [b, kv heads, groups, n, t]."""
    b, h, n, d = q.shape
    kv = h // groups
    s = torch.matmul(q.reshape(b, kv, groups * n, d) * scale, k.transpose(2, 3).contiguous()).view(b, kv, groups, n, -1)
    s = s.masked_fill_(~visible[:, None, None], -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp_(s.sub_(m))
    total = e.sum(dim=-1, keepdim=True)
    p = e.div_(torch.where(total > 0, total, 1.0))
    o = torch.matmul(p.view(b, kv, groups * n, -1), v)
    return o.reshape(b, h, n, d), (torch.log(total) + m).reshape(b, h, n), p


def _visible(at, keys, c, causal=True):
    """[b, n, t]: which keys the query at position `at` [b, n] sees"""
    t, p = torch.arange(keys, device="cuda"), at[:, :, None]
    see = (t <= p) if causal else torch.ones_like(t <= p)
    if c["window"]:
        see = see & ((p - t < c["window"]) | (t < c["sinks"]))
    return see


def _attention(s, c):
    if own:
        _device().attention(s["q"], s["k"], s["v"], causal=c["causal"], window=c["window"], sinks=c["sinks"], q_strides=s["q_strides"], k_strides=s["kv_strides"],
                            v_strides=s["kv_strides"], out=s["o"], out_strides=s["o_strides"])
        return s["seen"]["o"]
    q, k, v = _heads_apart(s["t"], c)
    at = torch.arange(c["queries"], device="cuda")[None] + (c["keys"] - c["queries"])
    o, _, _ = _weighted(q, k, v, _visible(at, c["keys"], c, c["causal"]), c["heads"] // c["kv_heads"], c["dim"] ** -0.5)
    return o.transpose(1, 2).to(TORCH[c["dtype"]]).contiguous()


def _rows_of(pages, table, longest):
    """the first `longest` rows of each sequence: [b, kv heads, longest, dim]"""
    n, g, page, d = pages.shape
    use = table[:, :-(-longest // page)].clamp(min=0).long()
    return pages[use].transpose(1, 2).reshape(use.shape[0], g, -1, d)[:, :, :longest]


def _paged(s, c):
    if own:
        extra = {"weights": s["weights"], "weights_out": s["weights_out"]} if c["weights"] else {}
        _device().paged_attention(s["q"], s["cache"], s["starts"], window=c["window"], sinks=c["sinks"], q_strides=s["strides"], out=s["o"], lse=s["lse"], **extra)
        return [s["seen"]["o"], s["seen"]["lse"]] + ([s["seen"]["weights_out"]] if c["weights"] else [])
    t, longest, most = s["t"], s["longest"], s["most"]
    lens, starts = t["lens"].long(), t["starts"].long()
    new = starts[1:] - starts[:-1]
    q, j = t["qkv"][:, :c["heads"]].float(), torch.arange(most, device="cuda")
    padded = q[(starts[:-1, None] + j).clamp(max=q.shape[0] - 1)].transpose(1, 2)               # [b, heads, most, dim]
    see = _visible((lens - new)[:, None] + j, longest, c) & (j < new[:, None])[:, :, None]
    k, v = _rows_of(t["k_pages"], t["table"], longest).float(), _rows_of(t["v_pages"], t["table"], longest).float()
    o, lse, p = _weighted(padded, k, v, see, c["heads"] // c["kv_heads"], c["dim"] ** -0.5)
    token = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    row = token - starts[seq]
    out = [o[seq, :, row].to(TORCH[c["dtype"]]), lse[seq, :, row]]
    if c["weights"]:
        at = torch.arange(longest, device="cuda")
        old = torch.where(at < (lens - new)[:, None, None], t["weights"][:, :, :longest], 0.0)
        t["weights_out"][:, :, :longest] = torch.where(at < lens[:, None, None], old + p.sum(dim=(2, 3)), t["weights_out"][:, :, :longest])
        out.append(t["weights_out"])
    return out


def _append(s, c):
    if own:
        _device().paged_append(s["cache"], s["starts"], s["k"], s["v"], k_strides=s["strides"], v_strides=s["strides"])
        return [s["seen"]["k_pages"], s["seen"]["v_pages"]]
    t, h, g = s["t"], c["heads"], c["kv_heads"]
    lens, starts = t["lens"].long(), t["starts"].long()
    token = torch.arange(t["qkv"].shape[0], device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    at = lens[seq] - starts[seq + 1] + token
    page, slot = t["table"][seq, at // c["page"]].long(), at % c["page"]
    t["k_pages"][page, :, slot] = t["qkv"][:, h:h + g]
    t["v_pages"][page, :, slot] = t["qkv"][:, h + g:]
    return [t["k_pages"], t["v_pages"]]


def _evict(s, c):
    if own:
        _device().paged_evict(s["cache"], s["weights"], c["keep"], first=c["first"], recent=c["recent"], to=s["to"], lens_out=s["lens_out"], weights_out=s["weights_out"])
        return [s["seen"][k] for k in ("k_pages", "v_pages", "weights_out", "lens_out")]
    t, longest, keep, page = s["t"], s["longest"], c["keep"], c["page"]
    lens, at = t["lens"].long(), torch.arange(s["longest"], device="cuda")
    here = at < lens[:, None, None]
    w = torch.where(here, t["weights"][:, :, :longest], -1.0)
    w = torch.where((at < c["first"]) | (at >= (lens - c["recent"])[:, None, None]) & here, math.inf, w)
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :, :keep]             # equal weights: the lower index first
    best = torch.sort(torch.where(best < lens[:, None, None], best, longest), dim=-1).values     # in order of position, what is not there last
    b, g, kept = best.shape
    target = torch.arange(kept, device="cuda")
    real = target < lens.clamp(max=keep)[:, None, None].expand(b, g, kept)
    best = torch.where(real, best, 0)
    seq, head = torch.arange(b, device="cuda")[:, None, None], torch.arange(g, device="cuda")[None, :, None]
    src, dst = t["table"].clamp(min=0).long()[seq, best // page], t["to"].clamp(min=0).long()[seq, (target // page)[None, None]]
    src_at, dst_at = (src * g + head) * page + best % page, (dst * g + head) * page + target % page
    # rows beyond a sequence's end go where the first one goes, with its value
    src_at, dst_at = torch.where(real, src_at, src_at[:, :, :1]), torch.where(real, dst_at, dst_at[:, :, :1])
    t["k_pages"].view(-1, c["dim"])[dst_at] = t["k_pages"].view(-1, c["dim"])[src_at]
    t["v_pages"].view(-1, c["dim"])[dst_at] = t["v_pages"].view(-1, c["dim"])[src_at]
    t["weights_out"][:, :, :kept] = torch.where(real, torch.gather(t["weights"][:, :, :longest], 2, best), t["weights_out"][:, :, :kept])
    t["lens_out"].copy_(lens.clamp(max=keep))
    return [t["k_pages"], t["v_pages"], t["weights_out"], t["lens_out"]]


# ---------------------------------------------------------------------------------------------------------- work, exact
def _pairs(length, new, window, sinks, causal=True):
    """visible (query, key) pairs of the last `new` of `length` tokens, and the keys that at least one of them sees"""
    if not causal:
        return new * length, length
    p = np.arange(max(0, length - new), length, dtype=np.int64)
    if not window:
        return int((p + 1).sum()), length
    inside = np.minimum(p + 1, window)
    first = p + 1 - inside
    return int((inside + np.minimum(sinks, first)).sum()), int(length - first[0] + min(sinks, first[0])) if len(p) else 0


def work(case):
    """each input read once (of the cache the rows that some query sees), each output written once; 4 flops a visible pair and column"""
    c, e = case, BYTES[case["dtype"]]
    row = c["kv_heads"] * c["dim"] * e
    if c["kind"] == "attention":
        pairs, keys = _pairs(c["keys"], c["queries"], c["window"], c["sinks"], c["causal"])
        return {"bytes": float(c["batch"] * (2 * keys * row + 2 * c["queries"] * c["heads"] * c["dim"] * e)), "flops": 4.0 * c["dim"] * c["batch"] * c["heads"] * pairs}
    lens, new = _lengths(c)
    if c["kind"] == "append":
        return {"bytes": float(4 * int(new.sum()) * row + 4 * int(new.sum())), "flops": 0.0}
    if c["kind"] == "evict":
        kept = np.minimum(lens, c["keep"])
        return {"bytes": float(4 * int(kept.sum()) * row + 4 * c["kv_heads"] * int((lens + kept).sum())), "flops": 0.0}
    both = [_pairs(int(n), int(m), c["window"], c["sinks"]) for n, m in zip(lens, new)]
    weights = 4 * c["kv_heads"] * (int(lens.sum()) + int((lens - new).sum())) if c["weights"] else 0
    tokens = int(new.sum())
    return {"bytes": float(2 * row * sum(k for _, k in both) + 2 * tokens * c["heads"] * c["dim"] * e + 4 * tokens * c["heads"] + weights),
            "flops": (4.0 * c["dim"] + (1 if c["weights"] else 0)) * c["heads"] * sum(p for p, _ in both)}


def _exact_head(q, k, v, at, c, causal=True):
    """one head in 64 bits, from the definition: o [n, d], lse [n], the weights [n, t]"""
    z = (q.double() @ k.double().T) / math.sqrt(c["dim"])
    t, p = torch.arange(k.shape[0], device="cuda")[None, :], at[:, None]
    hidden = torch.zeros_like(z, dtype=torch.bool)
    if causal:
        hidden |= t > p
    if c["window"]:
        hidden |= (t <= p - c["window"]) & (t >= c["sinks"])
    z[hidden] = -math.inf
    lse = torch.logsumexp(z, dim=1)
    w = torch.exp(z - lse[:, None])
    w[torch.isinf(lse)] = 0.0
    return w @ v.double(), lse, w


def exact(case, seed):
    c = case
    if c["kind"] not in ("attention", "paged"):
        return None                                             # nothing is computed there: values are moved
    t, groups = _inputs(c, seed), c["heads"] // c["kv_heads"]
    if c["kind"] == "attention":
        if "qkv" in t:
            q, k, v = t["qkv"][:, :, :c["heads"]], t["qkv"][:, :, c["heads"]:c["heads"] + c["kv_heads"]], t["qkv"][:, :, c["heads"] + c["kv_heads"]:]
        else:
            q, k, v = t["q"], t["k"], t["v"]
        o = torch.zeros(t["o"].shape, dtype=torch.float64, device="cuda")
        at = torch.arange(c["keys"] - c["queries"], c["keys"], device="cuda")
        for b in range(c["batch"]):
            for h in range(c["heads"]):
                o[b, :, h] = _exact_head(q[b, :, h], k[b, :, h // groups], v[b, :, h // groups], at, c, c["causal"])[0]
        return o
    lens, starts = t["lens"].tolist(), t["starts"].tolist()
    o = torch.zeros(t["o"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(o.shape[:2], dtype=torch.float64, device="cuda")
    w_out = torch.zeros(t["weights_out"].shape, dtype=torch.float64, device="cuda") if c["weights"] else None
    for b, length in enumerate(lens):
        first, last = starts[b], starts[b + 1]
        pages = t["table"][b, :-(-length // c["page"])].long()
        k, v = (t[x][pages].transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :length] for x in ("k_pages", "v_pages"))
        old = length - (last - first)
        at = torch.arange(old, length, device="cuda")
        for h in range(c["heads"]):
            o[first:last, h], lse[first:last, h], w = _exact_head(t["qkv"][first:last, h], k[h // groups], v[h // groups], at, c)
            if c["weights"]:
                w_out[b, h // groups, :length] += w.sum(dim=0)
        if c["weights"]:
            w_out[b, :, :old] += t["weights"][b, :, :old].double()
    return [o, lse] + ([w_out] if c["weights"] else [])
