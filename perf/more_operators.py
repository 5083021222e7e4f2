"""Cases of the operators between a projection and the next token: rotary positions of ragged tokens (alone, and with the rotated keys
and the values going to the pages of the cache), attention whose scores are capped, biased by distance or masked by documents and prefixes, and
sampling of tokens.

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
MOST_ROTATED = 5.4e7       # elements of q, k and v
MOST_LOGITS = 8.3e6

_open = {}


def _device():
    if "dev" not in _open:
        from ratchet_amd import Device
        _open["dev"] = Device(0)
    return _open["dev"]


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the next tokens of 64 conversations, queries and keys of one layer, pairs of neighbours rotated: the smallest call
        {"name": "rope_tokens_64_bf16", "kind": "rope", "dtype": "bf16", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": True,
         "farthest": 32768, "scaled": 0},
        # queries and keys of an 8192-token Phi-3 prompt that begins far into a long context, frequencies scaled by 32
        {"name": "rope_prompt_phi3_f16", "kind": "rope", "dtype": "f16", "tokens": 8192, "heads": 32, "kv_heads": 32, "dim": 96, "rotary": 96, "interleaved": False,
         "farthest": 131072, "scaled": 32},
        # a serving step of Phi-2, 32 of a head's 80 columns rotated: pieces of four prompts of up to 250 tokens next to twelve generated tokens
        {"name": "rope_append_step_phi2_f16", "kind": "rope_append", "dtype": "f16", "seqs": 16, "chunks": 4, "chunk": 250, "shortest": 300, "longest": 2000,
         "heads": 32, "kv_heads": 32, "dim": 80, "rotary": 32, "interleaved": False, "scaled": 0, "page": 32, "mix": 1},
        # one token for each of 64 long conversations: latency of a step
        {"name": "rope_append_tokens_64_bf16", "kind": "rope_append", "dtype": "bf16", "seqs": 64, "chunks": 0, "chunk": 0, "shortest": 200, "longest": 8000,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": True, "scaled": 8, "page": 16, "mix": 2},
        # a 4096-token prompt, scores capped at 50, a sliding window
        {"name": "prompt_cap_f16", "kind": "attention", "dtype": "f16", "batch": 1, "heads": 16, "kv_heads": 8, "dim": 256, "queries": 4096, "keys": 4096, "causal": True,
         "window": 2048, "sinks": 0, "cap": 50.0, "bias": False, "documents": 0, "prefix": 0, "mix": 3},
        # a 2048-token prompt whose scores fall with the distance
        {"name": "prompt_bias_bf16", "kind": "attention", "dtype": "bf16", "batch": 1, "heads": 32, "kv_heads": 32, "dim": 128, "queries": 2048, "keys": 2048, "causal": True,
         "window": 0, "sinks": 0, "cap": 0.0, "bias": True, "documents": 0, "prefix": 0, "mix": 4},
        # twelve texts packed into one row of 8192 tokens: the largest case
        {"name": "packed_documents_bf16", "kind": "attention", "dtype": "bf16", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "queries": 8192, "keys": 8192,
         "causal": True, "window": 0, "sinks": 0, "cap": 0.0, "bias": False, "documents": 12, "prefix": 0, "mix": 5},
        # Moondream's text model over two prompts: 729 image tokens that all see each other, then text
        {"name": "prompt_prefix_moondream_f16", "kind": "attention", "dtype": "f16", "batch": 2, "heads": 32, "kv_heads": 32, "dim": 64, "queries": 1100, "keys": 1100,
         "causal": True, "window": 0, "sinks": 0, "cap": 0.0, "bias": False, "documents": 0, "prefix": 730, "mix": 6},
        # one token for each of 32 conversations, scores capped and falling with the distance
        {"name": "tokens_32_cap_bias_bf16", "kind": "paged", "dtype": "bf16", "seqs": 32, "chunks": 0, "chunk": 0, "shortest": 200, "longest": 6000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "sinks": 0, "cap": 30.0, "bias": True, "prefix": 0, "mix": 7},
        # one token of a Whisper transcript, temperature alone: latency
        {"name": "sample_1_whisper_f32", "kind": "sample", "dtype": "f32", "rows": 1, "vocab": 51865, "padding": 0, "top_k": 0, "top_p": 1.0, "min_p": 0.0},
        # a step of 64 Phi-2 conversations, every filter in use, the logits as the last product pads them
        {"name": "sample_64_phi2_f16", "kind": "sample", "dtype": "f16", "rows": 64, "vocab": 50295, "padding": 905, "top_k": 50, "top_p": 0.95, "min_p": 0.02},
        # a step of 256 Phi-3 conversations, the nucleus alone
        {"name": "sample_256_phi3_f32", "kind": "sample", "dtype": "f32", "rows": 256, "vocab": 32064, "padding": 0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
    ]


def _spread(rng, low, high):
    """log-uniform over [low, high]"""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    while True:
        kind = rng.choice(["rope", "rope_append", "attention", "attention", "paged", "sample", "sample"])
        c = {"kind": kind, "dtype": rng.choice(["f16", "bf16", "f16", "bf16", "f32"])}
        heads, kv_heads = rng.choice([(6, 6), (8, 8), (32, 32), (32, 8), (16, 2), (12, 4), (16, 8)])
        dim, page, mix = rng.choice([64, 80, 96, 128, 40, 256]), rng.choice([16, 32, 64, 24, 128]), rng.randint(10, 10 ** 6)
        if kind == "sample":
            c.update(rows=_spread(rng, 1, 512), vocab=_spread(rng, 1000, 131072), padding=rng.choice([0, rng.randint(1, 1000)]), top_k=rng.choice([0, 1, _spread(rng, 2, 1000)]),
                     top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]))
        elif kind in ("rope", "rope_append"):
            c.update(heads=heads, kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, max(8, dim // 2 // 8 * 8), 32]), interleaved=rng.random() < 0.5, scaled=rng.choice([0, 4, 32]))
            if kind == "rope":
                c.update(tokens=_spread(rng, 1, 16384), farthest=_spread(rng, 100, 1 << 20))
        if kind in ("rope_append", "paged"):
            seqs, longest = _spread(rng, 1, 64), _spread(rng, 16, 8000)
            chunks = rng.choice([0, seqs, rng.randint(0, seqs)])
            c.update(seqs=seqs, chunks=chunks, chunk=_spread(rng, 2, 2048) if chunks else 0, shortest=rng.randint(1, longest), longest=longest, heads=heads, kv_heads=kv_heads,
                     dim=dim, page=page, mix=mix)
        if kind in ("attention", "paged"):
            window = rng.choice([0, 0, _spread(rng, 16, 4096)])
            c.update(heads=heads, kv_heads=kv_heads, dim=dim, window=window, sinks=rng.choice([0, rng.randint(1, 64)]) if window else 0, mix=mix,
                     cap=rng.choice([0.0, 20.0, 50.0]), bias=rng.random() < 0.4, prefix=rng.choice([0, 0, _spread(rng, 1, 1500)]))
        if kind == "attention":
            causal, queries = rng.random() < 0.8, rng.choice([1, _spread(rng, 2, 6000), _spread(rng, 2, 6000)])
            c.update(batch=_spread(rng, 1, 8), queries=queries, keys=queries if rng.random() < 0.7 else _spread(rng, queries, 8000), causal=causal,
                     documents=rng.choice([0, _spread(rng, 1, 40)]))
            if not causal:
                c.update(window=0, sinks=0, prefix=0)
        if kind in ("attention", "paged") and not (c["cap"] or c["bias"] or c["prefix"] or c.get("documents")):
            continue
        if _fits(c):
            return c


def _fits(c):
    if c["kind"] == "sample":
        return c["rows"] * c["vocab"] <= MOST_LOGITS
    if c["kind"] == "rope":
        return c["rotary"] <= c["dim"] and c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"] <= MOST_ROTATED
    if c["kind"] == "attention":
        return c["batch"] * c["heads"] * c["queries"] * c["keys"] <= MOST_SCORES
    lens, new = _lengths(c)
    if 2 * len(lens) * c["kv_heads"] * int(lens.max()) * c["dim"] * BYTES[c["dtype"]] > MOST_BYTES:
        return False
    if c["kind"] == "rope_append":
        return c["rotary"] <= c["dim"] and int(new.sum()) * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] <= MOST_ROTATED
    return len(lens) * c["heads"] * int(new.max()) * int(lens.max()) <= MOST_SCORES


def _lengths(c):
    """tokens in the cache of each sequence, the new ones among them, and how many are new"""
    r = np.random.RandomState(c["mix"])
    lens = r.randint(c["shortest"], c["longest"] + 1, c["seqs"])
    lens[r.randint(c["seqs"])] = c["longest"]
    new = np.ones_like(lens)
    if c["chunks"]:
        at = r.permutation(c["seqs"])[:c["chunks"]]
        new[at] = r.randint(max(1, c["chunk"] // 2), c["chunk"] + 1, c["chunks"])
        new[at[0]] = c["chunk"]
        lens = np.maximum(lens, new)
    return lens, new


def _documents(c):
    """[batch, documents + 1]: where each text begins and the last one ends; the rows after it are padding"""
    r, n = np.random.RandomState(c["mix"] + 1), c["documents"]
    out = np.zeros((c["batch"], n + 1), np.int64)
    for b in range(c["batch"]):
        end = c["keys"] if b == 0 else r.randint(c["keys"] * 3 // 4, c["keys"] + 1)
        out[b, 1:] = np.sort(np.concatenate([r.randint(0, end + 1, n - 1), [end]]))
    return out


def _prefixes(c):
    """tokens that all queries see: of each entry or sequence, of each of its documents where there are some"""
    r = np.random.RandomState(c["mix"] + 2)
    shape = (c["seqs"],) if c["kind"] == "paged" else (c["batch"], c["documents"]) if c["documents"] else (c["batch"],)
    out = r.randint(0, c["prefix"] + 1, shape)
    out.flat[0] = c["prefix"]
    return out


def _divisors(c):
    """what each frequency is divided by: long waves, which turn less than once in the context of the training, by the whole scale, short ones not at all"""
    if not c["scaled"]:
        return None
    f = 10000.0 ** (-2.0 * np.arange(c["rotary"] // 2) / c["rotary"])
    share = np.clip((4096 * f / (2 * math.pi) - 1) / (32 - 1), 0, 1)
    return 1.0 / (share + (1 - share) / c["scaled"])


def _factor(c):
    return 0.1 * math.log(c["scaled"]) + 1 if c["scaled"] else 1.0


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

    def normal(*shape, spread=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * spread).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32)

    def ints(v):
        return torch.as_tensor(np.ascontiguousarray(v, dtype=np.int32), device="cuda")

    if kind == "sample":
        # many unlikely tokens and a few likely ones, the more so the surer the model is of a row; a tenth of the rows is greedy
        rows, vocab = c["rows"], c["vocab"]
        x = torch.randn((rows, vocab), generator=gen, device="cuda") * 2.2 - 4
        likely = torch.randint(0, vocab, (rows, 24), generator=gen, device="cuda")
        x.scatter_(1, likely, torch.randn((rows, 24), generator=gen, device="cuda") * 2 + 14 * uniform(rows, 1))
        t = {"logits": torch.zeros(rows, vocab + c["padding"], device="cuda", dtype=dtype)}
        t["logits"][:, :vocab] = x.to(dtype)
        t["uniform"] = uniform(rows)
        t["temperature"] = torch.where(uniform(rows) < (0.1 if rows > 1 else 0.0), torch.zeros(rows, device="cuda"), 0.5 + uniform(rows))
        if c["top_k"]:
            t["top_k"] = ints(torch.randint(1, 2 * c["top_k"] + 1, (rows,), generator=gen, device="cuda").cpu()) if rows > 1 else ints([c["top_k"]])
        if c["top_p"] < 1:
            t["top_p"] = c["top_p"] + (1 - c["top_p"]) * uniform(rows) * 0.8
        if c["min_p"]:
            t["min_p"] = c["min_p"] * 2 * uniform(rows)
        t["tokens"], t["probs"] = torch.zeros(rows, device="cuda", dtype=torch.int32), torch.zeros(rows, device="cuda")
        return t
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    if kind == "rope":
        # q, k and v of a token side by side, as the projection leaves them; positions of a step in no order, those of a prompt one after the other
        n = c["tokens"]
        t = {"qkv": normal(n, h + 2 * g, d)}
        if n > 1024:
            t["positions"] = ints(max(0, c["farthest"] - n) + np.arange(n))
        else:
            t["positions"] = torch.randint(0, c["farthest"], (n,), generator=gen, device="cuda").to(torch.int32)
        t["o"] = torch.zeros(n, h + g, d, device="cuda", dtype=dtype)
        return t
    if kind == "attention":
        b, n, k = c["batch"], c["queries"], c["keys"]
        t = {"q": normal(b, n, h, d, spread=2.0), "k": normal(b, k, g, d), "v": normal(b, k, g, d)}
        if n == k:                                              # side by side, as one projection leaves them
            t = {"qkv": torch.cat([t["q"], t["k"], t["v"]], dim=2)}
        t["o"], t["lse"] = torch.zeros(b, n, h, d, device="cuda", dtype=dtype), torch.zeros(b, h, n, device="cuda")
        if c["documents"]:
            t["documents"] = ints(_documents(c))
    else:
        lens, new = _lengths(c)
        page = c["page"]
        each = -(-lens // page)                                 # pages of each sequence
        total, width = int(each.sum()) + 3, int(each.max()) + 2
        order = np.random.RandomState(int(seed) % (1 << 31)).permutation(total)
        table = np.full((len(lens), width), -1, np.int64)
        for i, at in enumerate(np.concatenate([[0], np.cumsum(each)])[:-1]):
            table[i, :each[i]] = order[at:at + each[i]]
        tokens = int(new.sum())
        t = {"k_pages": normal(total, g, page, d), "v_pages": normal(total, g, page, d), "table": ints(table), "lens": ints(lens),
             "starts": ints(np.concatenate([[0], np.cumsum(new)]))}
        t["qkv"] = torch.cat([normal(tokens, h, d, spread=2.0), normal(tokens, 2 * g, d)], dim=1)
        t["o"] = torch.zeros(tokens, h, d, device="cuda", dtype=dtype)
        if kind == "rope_append":
            return t
        t["lse"] = torch.zeros(tokens, h, device="cuda")
    if c["bias"]:
        t["slopes"] = torch.as_tensor(2.0 ** (-8.0 * np.arange(1, h + 1) / h), device="cuda").float()
    if c["prefix"]:
        t["prefix"] = ints(_prefixes(c))
    return t


def prepare(case, seed):
    c, t = case, _inputs(case, seed)
    s = {"case": c}
    if "seqs" in c:
        lens, new = _lengths(c)
        s["longest"], s["most"] = int(lens.max()), int(new.max())
    if "rotary" in c:
        s["factor"] = _factor(c)
    if not own:
        if "rotary" in c:
            f = 10000.0 ** (-2.0 * np.arange(c["rotary"] // 2) / c["rotary"])
            t["frequencies"] = torch.as_tensor(f / _divisors(c) if c["scaled"] else f, device="cuda")
        s["t"] = t
        return s
    dev, both = _device(), {k: _buffer(v) for k, v in t.items()}
    b, s["seen"] = {k: v[0] for k, v in both.items()}, {k: v[1] for k, v in both.items()}
    if "rotary" in c:
        s["turns"] = dev.rope_table(c["rotary"], 10000.0, _divisors(c))
    s.update(b)
    if c["kind"] == "sample":
        s["logits"], s["stride"] = b["logits"].view(0, (c["rows"], c["vocab"])), c["vocab"] + c["padding"]
        return s
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    w, at = h + 2 * g, (0, h * d, (h + g) * d)                  # q, k and v are windows of the projection's rows
    if c["kind"] == "attention":
        n, k = c["queries"], c["keys"]
        if "qkv" in b:
            s["q"], s["k"], s["v"] = (b["qkv"].view(o, (c["batch"], x, n, d)) for o, x in zip(at, (h, g, g)))
            s["q_strides"] = s["kv_strides"] = (n * w * d, d, w * d, 1)
        else:
            s["q"], s["k"], s["v"] = b["q"].reshape((c["batch"], h, n, d)), b["k"].reshape((c["batch"], g, k, d)), b["v"].reshape((c["batch"], g, k, d))
            s["q_strides"], s["kv_strides"] = (n * h * d, d, h * d, 1), (k * g * d, d, g * d, 1)
        s["o"], s["o_strides"] = b["o"].reshape((c["batch"], h, n, d)), (n * h * d, d, h * d, 1)
        return s
    n, s["strides"] = b["qkv"].shape[0], (w * d, d)
    s["q"], s["k"], s["v"] = (b["qkv"].view(o, (n, x, d)) for o, x in zip(at, (h, g, g)))
    if c["kind"] == "rope":
        s["qk"] = b["qkv"].view(0, (n, h + g, d))
    else:
        s["cache"] = dev.paged_cache(b["k_pages"], b["v_pages"], b["table"], b["lens"])
    return s


# ----------------------------------------------------------------------------------------------------------------- run
def run(state):
    c = state["case"]
    return {"rope": _rope, "rope_append": _rope_append, "attention": _attention, "paged": _paged, "sample": _sample}[c["kind"]](state, c)


def _rotate(x, positions, frequencies, factor, interleaved, dtype):
    """x [tokens, heads, dim] at `positions`: angles in 64 bits, as 32 do not hold those of far positions, the rest in 32"""
    angle = positions.double()[:, None] * frequencies
    cos, sin = (torch.cos(angle) * factor).float()[:, None], (torch.sin(angle) * factor).float()[:, None]
    half = frequencies.shape[0]
    y = x.float()
    turned, rest = y[..., :2 * half], y[..., 2 * half:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    one, two = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([one, two], dim=-1).flatten(-2) if interleaved else torch.cat([one, two], dim=-1)
    return torch.cat([turned, rest], dim=-1).to(dtype)


def _rope(s, c):
    if own:
        _device().rope_tokens(s["qk"], s["positions"], s["turns"], factor=s["factor"], interleaved=c["interleaved"], strides=s["strides"], out=s["o"])
        return s["seen"]["o"]
    t = s["t"]
    return _rotate(t["qkv"][:, :c["heads"] + c["kv_heads"]], t["positions"], t["frequencies"], s["factor"], c["interleaved"], TORCH[c["dtype"]])


def _rope_append(s, c):
    if own:
        _device().paged_rope_append(s["cache"], s["starts"], s["q"], s["k"], s["v"], s["turns"], factor=s["factor"], interleaved=c["interleaved"], q_strides=s["strides"],
                                    k_strides=s["strides"], v_strides=s["strides"], out=s["o"])
        return [s["seen"][k] for k in ("o", "k_pages", "v_pages")]
    t, h, g = s["t"], c["heads"], c["kv_heads"]
    lens, starts = t["lens"].long(), t["starts"].long()
    token = torch.arange(t["qkv"].shape[0], device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    at = lens[seq] - starts[seq + 1] + token
    turned = _rotate(t["qkv"][:, :h + g], at, t["frequencies"], s["factor"], c["interleaved"], TORCH[c["dtype"]])
    page, slot = t["table"][seq, at // c["page"]].long(), at % c["page"]
    t["k_pages"][page, :, slot] = turned[:, h:]
    t["v_pages"][page, :, slot] = t["qkv"][:, h + g:]
    return [turned[:, :h].contiguous(), t["k_pages"], t["v_pages"]]


def _weighted(q, k, v, visible, distance, slopes, c):
    """softmax of the changed scores times v, in 32 bits: q [b, heads, n, d], k and v [b, kv heads, t, d], visible [b, n, t], distance
    [b or 1, n, t].  Returns o [b, heads, n, d] and lse [b, heads, n]."""
    b, h, n, d = q.shape
    kv = k.shape[1]
    s = torch.matmul(q.reshape(b, kv, h // kv * n, d) * d ** -0.5, k.transpose(2, 3).contiguous()).view(b, kv, h // kv, n, -1)
    if c["cap"]:
        s = s.div_(c["cap"]).tanh_().mul_(c["cap"])
    if c["bias"]:
        s = s.sub_(slopes.view(1, kv, h // kv, 1, 1) * distance[:, None, None])
    s = s.masked_fill_(~visible[:, None, None], -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp_(s.sub_(m))
    total = e.sum(dim=-1, keepdim=True)
    p = e.div_(torch.where(total > 0, total, 1.0))
    o = torch.matmul(p.view(b, kv, h // kv * n, -1), v)
    return o.reshape(b, h, n, d), (torch.log(total) + m).reshape(b, h, n)


def _visible(at, keys, c, low, high, prefix):
    """[b, n, t]: which keys the query at position `at` [b, n] sees; low, high and prefix [b, n]: its document, and how much of it all queries see"""
    t, p, low = torch.arange(keys, device="cuda"), at[:, :, None], low[:, :, None]
    see = (t >= low) & (t < high[:, :, None])
    if c.get("causal", True):
        back = t <= p
        if c["window"]:
            back = back & ((p - t < c["window"]) | (t - low < c["sinks"]))
        see = see & (back | (t - low < prefix[:, :, None]))
    return see


def _attention(s, c):
    if own:
        _device().attention(s["q"], s["k"], s["v"], causal=c["causal"], window=c["window"], sinks=c["sinks"], q_strides=s["q_strides"], k_strides=s["kv_strides"],
                            v_strides=s["kv_strides"], out=s["o"], out_strides=s["o_strides"], lse=s["lse"], cap=c["cap"], slopes=s.get("slopes"), documents=s.get("documents"),
                            prefix=s.get("prefix"))
        return [s["seen"]["o"], s["seen"]["lse"]]
    t, h, g = s["t"], c["heads"], c["kv_heads"]
    q, k, v = t["qkv"].split([h, g, g], dim=2) if "qkv" in t else (t["q"], t["k"], t["v"])
    q, k, v = (x.transpose(1, 2).float() for x in (q, k, v))
    at = (torch.arange(c["queries"], device="cuda") + (c["keys"] - c["queries"])).expand(c["batch"], -1).contiguous()
    low, high, prefix = torch.zeros_like(at), torch.full_like(at, c["keys"]), torch.zeros_like(at)
    if c["documents"]:
        doc = torch.searchsorted(t["documents"].long(), at, right=True) - 1            # of each query's position
        inside = (doc >= 0) & (doc < c["documents"])
        doc = doc.clamp(0, c["documents"] - 1)
        low, high = t["documents"].long().gather(1, doc), t["documents"].long().gather(1, doc + 1)
        high = torch.where(inside, high, low)
        if c["prefix"]:
            prefix = t["prefix"].long().gather(1, doc)
    elif c["prefix"]:
        prefix = t["prefix"].long()[:, None].expand_as(at)
    distance = (at[0, :, None] - torch.arange(c["keys"], device="cuda")).abs().float()[None]
    o, lse = _weighted(q, k, v, _visible(at, c["keys"], c, low, high, prefix), distance, t.get("slopes"), c)
    return [o.transpose(1, 2).to(TORCH[c["dtype"]]).contiguous(), lse]


def _rows_of(pages, table, longest):
    """the first `longest` rows of each sequence: [b, kv heads, longest, dim]"""
    n, g, page, d = pages.shape
    use = table[:, :-(-longest // page)].clamp(min=0).long()
    return pages[use].transpose(1, 2).reshape(use.shape[0], g, -1, d)[:, :, :longest]


def _paged(s, c):
    if own:
        _device().paged_attention(s["q"], s["cache"], s["starts"], window=c["window"], sinks=c["sinks"], q_strides=s["strides"], out=s["o"], lse=s["lse"], cap=c["cap"],
                                  slopes=s.get("slopes"), prefix=s.get("prefix"))
        return [s["seen"]["o"], s["seen"]["lse"]]
    t, longest, most = s["t"], s["longest"], s["most"]
    lens, starts = t["lens"].long(), t["starts"].long()
    new = starts[1:] - starts[:-1]
    q, j = t["qkv"][:, :c["heads"]].float(), torch.arange(most, device="cuda")
    padded = q[(starts[:-1, None] + j).clamp(max=q.shape[0] - 1)].transpose(1, 2)               # [b, heads, most, dim]
    at = (lens - new)[:, None] + j
    prefix = t["prefix"].long()[:, None].expand_as(at) if c["prefix"] else torch.zeros_like(at)
    see = _visible(at, longest, c, torch.zeros_like(at), lens[:, None].expand_as(at), prefix) & (j < new[:, None])[:, :, None]
    k, v = _rows_of(t["k_pages"], t["table"], longest).float(), _rows_of(t["v_pages"], t["table"], longest).float()
    distance = (at[:, :, None] - torch.arange(longest, device="cuda")).abs().float()
    o, lse = _weighted(padded, k, v, see, distance, t.get("slopes"), c)
    token = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    row = token - starts[seq]
    return [o[seq, :, row].to(TORCH[c["dtype"]]), lse[seq, :, row]]


def _sample(s, c):
    if own:
        _device().sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s.get("top_k"), top_p=s.get("top_p"), min_p=s.get("min_p"), row_stride=s["stride"],
                         out=s["tokens"], probs=s["probs"])
        return [s["seen"]["tokens"], s["seen"]["probs"]]
    # in 64 bits: the border between two tokens, and between a kept and a dropped one, decides about the answer
    t, vocab = s["t"], c["vocab"]
    x, order = torch.sort(t["logits"][:, :vocab].double(), dim=1, descending=True, stable=True)          # equal logits: the lower index first
    greedy = t["temperature"] <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, t["temperature"])[:, None].double())
    rank = torch.arange(vocab, device="cuda")[None]
    keep = torch.where(greedy, 1, t["top_k"].long() if "top_k" in t else vocab)[:, None]
    w = torch.where(rank < keep, w, 0.0)
    if "min_p" in t:
        enough = w >= t["min_p"].double()[:, None]
    if "top_p" in t:
        before = torch.cumsum(w, dim=1) - w
        w = torch.where(before < t["top_p"].double()[:, None] * w.sum(dim=1, keepdim=True), w, 0.0)
    if "min_p" in t:
        w = torch.where(enough, w, 0.0)
    total = w.sum(dim=1)
    upto = torch.cumsum(torch.zeros_like(w).scatter_(1, order, w), dim=1)
    token = (upto <= (t["uniform"].double() * upto[:, -1])[:, None]).sum(dim=1)
    mine = torch.zeros_like(w).scatter_(1, order, w).gather(1, token[:, None])[:, 0]
    return [token.to(torch.int32), (mine / total).float()]


# ---------------------------------------------------------------------------------------------------------- work, exact
def _pairs(length, new, c, low=0, high=None, prefix=0):
    """visible (query, key) pairs of the last `new` of the tokens [low, high) of which `length` - low are at hand, and the keys that one of them sees"""
    high = length if high is None else high
    p = np.arange(max(low, length - new), length, dtype=np.int64)
    p = p[(p >= low) & (p < high)]
    if not len(p):
        return 0, 0
    if not c.get("causal", True):
        return int(len(p) * (high - low)), int(high - low)
    last = np.maximum(p, min(low + prefix, high) - 1)           # the last key it sees
    if not c["window"]:
        return int((last + 1 - low).sum()), int(last[-1] + 1 - low)
    first = np.maximum(low, p - c["window"] + 1)                # of its window
    front = np.minimum(min(low + max(c["sinks"], prefix), high), first)                # what lies before the window
    beyond = np.maximum(0, last - np.maximum(p, first - 1))
    return int((p - first + 1 + front - low + beyond).sum()), int(last[-1] + 1 - first[0] + max(0, front[0] - low))


def work(case):
    """each input read once (of the cache the rows that some query sees), each output written once; 4 flops a visible pair and column, 4 a rotated column"""
    c, e = case, BYTES[case["dtype"]]
    if c["kind"] == "sample":
        filters = 8 + 4 * (bool(c["top_k"]) + (c["top_p"] < 1) + bool(c["min_p"])) + 8
        return {"bytes": float(c["rows"] * (c["vocab"] * e + filters)), "flops": 2.0 * c["rows"] * c["vocab"]}
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "rope":
        return {"bytes": float(c["tokens"] * (2 * (h + g) * d * e + 4)), "flops": 4.0 * c["tokens"] * (h + g) * c["rotary"]}
    row = g * d * e
    if c["kind"] == "attention":
        pairs = keys = 0
        docs = _documents(c) if c["documents"] else np.array([[0, c["keys"]]] * c["batch"])
        pre = np.zeros((c["batch"], docs.shape[1] - 1), np.int64) + (_prefixes(c).reshape(c["batch"], -1) if c["prefix"] else 0)
        for b in range(c["batch"]):
            for i in range(docs.shape[1] - 1):
                more = _pairs(c["keys"], c["queries"], c, int(docs[b, i]), int(docs[b, i + 1]), int(pre[b, i]))
                pairs, keys = pairs + more[0], keys + more[1]
        rows = c["batch"] * c["queries"] * h
        return {"bytes": float(2 * keys * row + rows * (2 * d * e + 4)), "flops": 4.0 * d * h * pairs}
    lens, new = _lengths(c)
    tokens = int(new.sum())
    if c["kind"] == "rope_append":
        return {"bytes": float(tokens * (2 * h * d * e + 4 * row + 4)), "flops": 4.0 * tokens * (h + g) * c["rotary"]}
    pre = _prefixes(c) if c["prefix"] else np.zeros(len(lens), np.int64)
    both = [_pairs(int(n), int(m), c, prefix=int(x)) for n, m, x in zip(lens, new, pre)]
    return {"bytes": float(2 * row * sum(k for _, k in both) + 2 * tokens * h * d * e + 4 * tokens * h), "flops": 4.0 * d * h * sum(p for p, _ in both)}


def _exact_turned(x, positions, c):
    """every pair as a complex number, turned by e^(i angle)"""
    half = c["rotary"] // 2
    f = np.array([10000.0 ** (-i / half) for i in range(half)])
    if c["scaled"]:
        f = f / _divisors(c)
    angle = positions.double()[:, None, None] * torch.as_tensor(f, device="cuda")
    turn = torch.polar(torch.full_like(angle, _factor(c)), angle)
    y = x.double().clone()
    one, two = (slice(0, c["rotary"], 2), slice(1, c["rotary"], 2)) if c["interleaved"] else (slice(0, half), slice(half, c["rotary"]))
    z = torch.complex(x[..., one].double(), x[..., two].double()) * turn
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _exact_head(q, k, v, at, c, h, low, high, prefix):
    """one head's queries of one document in 64 bits, from the definition: o [n, d], lse [n]"""
    z = (q.double() @ k[low:high].double().T) / math.sqrt(c["dim"])
    t, p = torch.arange(low, high, device="cuda")[None, :], at[:, None]
    if c["cap"]:
        z = c["cap"] * torch.tanh(z / c["cap"])
    if c["bias"]:
        z = z - float(np.float32(2.0 ** (-8.0 * (h + 1) / c["heads"]))) * (t - p).abs()
    if c.get("causal", True):
        hidden = t > p
        if c["window"]:
            hidden = hidden | ((t <= p - c["window"]) & (t >= low + c["sinks"]))
        z[hidden & (t >= low + prefix)] = -math.inf
    lse = torch.logsumexp(z, dim=1)
    w = torch.exp(z - lse[:, None])
    w[torch.isinf(lse)] = 0.0
    return w @ v[low:high].double(), lse


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    if c["kind"] == "sample":
        tokens, probs = [], []
        for r in range(c["rows"]):
            x = t["logits"][r, :c["vocab"]].double()
            temperature = float(t["temperature"][r])
            if temperature <= 0:
                tokens.append(int((x == x.max()).nonzero()[0, 0]))
                probs.append(1.0)
                continue
            w = torch.exp((x - x.max()) / temperature)
            order = torch.argsort(x, descending=True, stable=True)
            if "top_k" in t:
                order = order[:int(t["top_k"][r])]
            kept = len(order)
            if "top_p" in t:
                sums = torch.cumsum(w[order], 0)
                kept = 1 + int((sums < float(t["top_p"][r]) * float(sums[-1])).sum())
            if "min_p" in t:
                kept = min(kept, int((w[order] >= float(t["min_p"][r])).sum()))
            kept = torch.sort(order[:kept]).values
            sums = torch.cumsum(w[kept], 0)
            token = int(kept[int(torch.searchsorted(sums, float(t["uniform"][r]) * float(sums[-1]), right=True))])
            tokens.append(token)
            probs.append(float(w[token] / sums[-1]))
        return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)]
    h, g = c["heads"], c["kv_heads"]
    if c["kind"] == "rope":
        return _exact_turned(t["qkv"][:, :h + g], t["positions"], c)
    groups = h // g
    if c["kind"] == "attention":
        q, k, v = (t["qkv"][:, :, :h], t["qkv"][:, :, h:h + g], t["qkv"][:, :, h + g:]) if "qkv" in t else (t["q"], t["k"], t["v"])
        o = torch.zeros(t["o"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full(t["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
        docs = t["documents"].tolist() if c["documents"] else [[0, c["keys"]]] * c["batch"]
        pre = t["prefix"].reshape(c["batch"], -1).tolist() if c["prefix"] else [[0] * (len(docs[0]) - 1)] * c["batch"]
        first = c["keys"] - c["queries"]                        # position of row 0
        for b in range(c["batch"]):
            for low, high, prefix in zip(docs[b][:-1], docs[b][1:], pre[b]):
                r0, r1 = max(low - first, 0), min(high - first, c["queries"])
                if r0 >= r1:
                    continue
                at = torch.arange(first + r0, first + r1, device="cuda")
                for i in range(h):
                    o[b, r0:r1, i], lse[b, i, r0:r1] = _exact_head(q[b, r0:r1, i], k[b, :, i // groups], v[b, :, i // groups], at, c, i, low, high, prefix)
        return [o, lse]
    lens, starts = t["lens"].tolist(), t["starts"].tolist()
    if c["kind"] == "rope_append":
        at = torch.cat([torch.arange(n - (e - s), n, device="cuda") for n, s, e in zip(lens, starts[:-1], starts[1:])])
        turned = _exact_turned(t["qkv"][:, :h + g], at, c)
        k_pages = t["k_pages"].double()
        for b in range(len(lens)):
            for i in range(starts[b], starts[b + 1]):
                p = lens[b] - starts[b + 1] + i
                page = int(t["table"][b, p // c["page"]]) if (p % c["page"] == 0 or i == starts[b]) else page
                k_pages[page, :, p % c["page"]] = turned[i, h:]
        return [turned[:, :h], k_pages, None]                   # values are moved
    o = torch.zeros(t["o"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(o.shape[:2], dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        first, last = starts[b], starts[b + 1]
        pages = t["table"][b, :-(-length // c["page"])].long()
        k, v = (t[x][pages].transpose(0, 1).reshape(g, -1, c["dim"])[:, :length] for x in ("k_pages", "v_pages"))
        at = torch.arange(length - (last - first), length, device="cuda")
        for i in range(h):
            o[first:last, i], lse[first:last, i] = _exact_head(t["qkv"][first:last, i], k[i // groups], v[i // groups], at, c, i, 0, length, int(t["prefix"][b]) if c["prefix"] else 0)
    return [o, lse]
