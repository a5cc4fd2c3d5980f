"""The operators of a serving step with drafted tokens, as cases to be timed.

A program that serves a model with a draft (a tree of guessed tokens, checked in
one pass) makes these calls each step (include/mi_hip_attn.h):

  norm_rope   mi_hip_norm_rope_append: the norms of queries and keys per head
              (models that have them), the rotation at each token's own position,
              and the append of K and V to an F32, F16 or 8-bit cache, in one pass;
  cache       mi_hip_kv_write, mi_hip_kv_keep, mi_hip_kv_read on an 8-bit cache:
              rows quantised as they are written, the accepted rows of a tree
              moved together, rows read back;
  attn        mi_hip_attn_tree: attention of a tree of drafted tokens, of a causal
              chunk or of single tokens over such a cache, one or many sequences;
  logits      mi_hip_logits_adjust: penalties for repeated tokens, biases and
              grammar masks on the logits, and the greedy ids.

Shapes are the repository's own: 14/2 heads of 64 (Qwen2.5-0.5B), 28/4 heads of
128 (the 7B head shape), a vocabulary of 151936.

The 8-bit cache: a group's scale d is the smallest f16 number with 127 d >= max |x|
(a K row has a group for each 32 dims, a V row is one group), an element the whole
number nearest to x / d, ties to the even one.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

QWEN05B = dict(n_head=14, n_head_kv=2, head_dim=64)
QWEN7B = dict(n_head=28, n_head_kv=4, head_dim=128)
VOCAB = 151936
K_GROUP = 32


def _rope(n_tokens, n_past, cache, shape, norm=True, tree=False):
    return dict(kind="norm_rope", n_tokens=n_tokens, n_past=n_past, cache=cache, norm=norm, tree=tree, **shape)


def _cache(n_tokens, n_past, keep, out, shape):
    return dict(kind="cache", n_tokens=n_tokens, n_past=n_past, keep=keep, out=out, **shape)


def _attn(items, n_past, n_tokens, cache, tree, shape):
    return dict(kind="attn", items=items, n_past=n_past, n_tokens=n_tokens, cache=cache, tree=tree, **shape)


def _logits(rows, vocab, history, biases, grammar):
    return dict(kind="logits", rows=rows, vocab=vocab, history=history, biases=biases, grammar=grammar)


def listed():
    def named(name, c):
        return dict(c, name=name)
    return [
        # one generated token of a model with q/k norms, F32 cache: latency
        named("norm_rope_1_f32", _rope(1, 600, "f32", QWEN05B)),
        # a tree of drafted tokens at their depths' positions, 8-bit cache
        named("norm_rope_tree_25_q8", _rope(25, 2000, "q8", QWEN7B, tree=True)),
        # a prompt's chunk, F16 cache
        named("norm_rope_4096_f16", _rope(4096, 1337, "f16", QWEN7B)),
        # a tree's rows written to an 8-bit cache, the accepted ones kept and read
        named("cache_tree_25_keep_6", _cache(25, 1000, 6, "f32", QWEN05B)),
        # a long prefix put into an 8-bit cache and read back
        named("cache_16384", _cache(16384, 0, 0, "f16", QWEN7B)),
        # a small tree early in a chat, F32 cache: latency
        named("tree_8x519_f32", _attn(1, 511, 8, "f32", True, QWEN05B)),
        # one token of 24 sequences over 8-bit caches, ragged lengths
        named("decode_24x4096_q8", _attn(24, 4095, 1, "q8", False, QWEN05B)),
        # a tree of the 7B shape, F16 cache, odd sizes
        named("tree_25x4132_f16", _attn(1, 4107, 25, "f16", True, QWEN7B)),
        # a prompt's chunk over an 8-bit cache (the causal form)
        named("chunk_1024x2361_q8", _attn(1, 1337, 1024, "q8", False, QWEN05B)),
        # four sequences with wide trees over long 8-bit caches
        named("tree_4x64x16384_q8", _attn(4, 16320, 64, "q8", True, QWEN7B)),
        # one row of logits: a chat with a repetition penalty
        named("logits_1", _logits(1, VOCAB, 300, 0, False)),
        # every node of a batch's trees: penalties, biases and a grammar
        named("logits_64_grammar", _logits(64, VOCAB, 2048, 100, True)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_rope", "cache", "attn", "attn", "logits"])
    shape = rng.choice([QWEN05B, QWEN7B])
    if kind == "norm_rope":
        t = _log(rng, 1, 4096)
        return _rope(t, rng.choice([0, _log(rng, 1, 4096)]), rng.choice(["f32", "f16", "q8"]), shape,
                     norm=rng.random() < 0.7, tree=t <= 64 and rng.random() < 0.5)
    if kind == "cache":
        t = _log(rng, 1, 16384)
        return _cache(t, rng.choice([0, _log(rng, 1, 4096)]), rng.randint(1, min(t, 16)) if t <= 64 else 0,
                      rng.choice(["f32", "f16"]), shape)
    if kind == "logits":
        return _logits(_log(rng, 1, 64), rng.choice([VOCAB, _log(rng, 1000, VOCAB)]), rng.choice([0, _log(rng, 1, 2048)]),
                       rng.choice([0, _log(rng, 1, 100)]), rng.random() < 0.5)
    tree = rng.random() < 0.6
    t = _log(rng, 1, 64) if tree or rng.random() < 0.5 else _log(rng, 64, 1024)
    past = _log(rng, 16, 16384)
    items = rng.randint(1, 24) if rng.random() < 0.5 else 1
    # at most 2^22 (query, key) pairs and 2^17 keys over the items
    items = max(1, min(items, (1 << 22) // (t * (past + t)), (1 << 17) // (past + t)))
    past = max(16, min(past, (1 << 22) // t - t))
    return _attn(items, past, t, rng.choice(["f32", "f16", "q8"]), tree, shape)


# ---- inputs -------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tree(seed, n):
    """A random tree of n drafted tokens: depths, and each one's ancestors and itself as bits of 64-bit words."""
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    words = (n + 63) // 64
    seen, depth = [], np.zeros(n, dtype=np.int32)
    bits = np.zeros((n, words), dtype=np.uint64)
    for i in range(n):
        parent = rng.randint(max(-1, i - 8), i) if i else -1
        seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        depth[i] = depth[parent] + 1 if parent >= 0 else 0
        for w in range(words):
            bits[i, w] = seen[i] >> 64 * w & 0xFFFFFFFFFFFFFFFF
    return depth, bits.view(np.int64)


def _quantise(x, group):
    """The 8-bit form of the rows of x (..., head_dim): int8 values and f16 scales (..., head_dim / group)."""
    g = x.view(*x.shape[:-1], -1, group)
    amax = g.abs().amax(-1).double()
    h = (amax / 127.0).to(torch.float16)
    bits = h.view(torch.int16)
    up = 127.0 * h.double() < amax
    down = (bits > 0) & (127.0 * (bits - 1).view(torch.float16).double() >= amax)
    d = (bits + up.to(torch.int16) - down.to(torch.int16)).view(torch.float16)
    q = torch.round(g.double() / torch.where(d > 0, d, torch.ones_like(d)).double()[..., None])
    return q.to(torch.int8).view(x.shape), d


def _values(q, d):
    """What the 8-bit form stands for, in 32 bits (exactly)."""
    group = q.shape[-1] // d.shape[-1]
    return (q.float().view(*d.shape, group) * d.float()[..., None]).view(q.shape)


def _keys(shape, g):
    """Rows of K before the cache: some channels are far larger than the rest."""
    k = torch.randn(shape, device="cuda", generator=g)
    k[..., ::29] *= 8.0
    return k


def _rope_inputs(case, seed):
    g = _gen(seed)
    t, h, hk, d = case["n_tokens"], case["n_head"], case["n_head_kv"], case["head_dim"]
    s = dict(q=torch.randn((t, h, d), device="cuda", generator=g) * 2.0, k=_keys((t, hk, d), g),
             v=torch.randn((t, hk, d), device="cuda", generator=g))
    if case["norm"]:
        s["q_norm"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
        s["k_norm"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
    s["freq"] = (1e6 ** (-np.arange(0, d, 2, dtype=np.float64) / d)).astype(np.float32)
    step = torch.from_numpy(_tree(seed, t)[0]) if case["tree"] else torch.arange(t, dtype=torch.int32)
    s["pos"] = (case["n_past"] + step).to(torch.int32).cuda()
    return s


def _cache_inputs(case, seed):
    g = _gen(seed)
    t, hk, d = case["n_tokens"], case["n_head_kv"], case["head_dim"]
    keep = np.sort(np.random.RandomState(seed & 0x7FFFFFFF).permutation(t)[:case["keep"]]).astype(np.int32)
    return dict(k=_keys((t, hk, d), g), v=torch.randn((t, hk, d), device="cuda", generator=g), keep=keep)


def _pasts(case):
    """Each sequence's cached positions: ragged, the first the longest."""
    n, past = case["items"], case["n_past"]
    return [past - i * past // (3 * n) for i in range(n)]


def _attn_inputs(case, seed):
    g = _gen(seed)
    n, t, d = case["items"], case["n_tokens"], case["head_dim"]
    n_ctx = case["n_past"] + t
    q = torch.randn((n, t, case["n_head"], d), device="cuda", generator=g)
    k = torch.randn((n, n_ctx, case["n_head_kv"], d), device="cuda", generator=g)
    v = torch.randn((n, n_ctx, case["n_head_kv"], d), device="cuda", generator=g)
    bits = torch.from_numpy(np.stack([_tree(seed + i, t)[1] for i in range(n)])).cuda() if case["tree"] else None
    return q, k, v, bits


def _logits_inputs(case, seed):
    g = _gen(seed)
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    rows, vocab = case["rows"], case["vocab"]
    s = dict(logits=torch.randn((rows, vocab), device="cuda", generator=g) * 3.0)
    # every row has its own request's penalties and a history of its own length
    s["penalties"] = torch.rand((rows, 3), device="cuda", generator=g) * torch.tensor([0.5, 0.3, 0.3], device="cuda")
    s["penalties"][:, 0] += 1.0
    lens = rng.randint(case["history"] // 2, case["history"] + 1, rows) if case["history"] else np.zeros(rows, np.int64)
    ids = np.minimum((rng.pareto(0.6, int(lens.sum())) * 50).astype(np.int64) % vocab, vocab - 1)
    s["hist"] = torch.from_numpy(ids.astype(np.int32)).cuda()
    s["hist_off"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()
    n = case["biases"]
    s["bias_id"] = torch.from_numpy(np.concatenate([rng.permutation(vocab)[:n] for _ in range(rows)]).astype(np.int32)).cuda()
    s["bias"] = torch.randn(rows * n, device="cuda", generator=g) * 4.0
    s["bias_off"] = torch.arange(rows + 1, dtype=torch.int32, device="cuda") * n
    s["mask"] = None
    if case["grammar"]:  # a third of the words of 32 tokens empty, random bits in the rest
        words = (vocab + 31) // 32
        m = torch.randint(-2**31, 2**31, (rows, words), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
        s["mask"] = m * (torch.rand((rows, words), device="cuda", generator=g) < 0.667)
    return s


# ---- what a user's program keeps of the framework -------------------------------


def _lib():
    where = os.path.join(os.getcwd(), "mini-infer-llama.cpp_amd")
    if where not in sys.path:
        sys.path.insert(1, where)
    import mi_hip_attn as mh
    torch.cuda.current_stream()  # torch's HIP runtime comes up first
    lib = mh.lib()
    lib.init(torch.cuda.current_device())
    return mh, lib


def _cache_type(mh, name):
    return {"f32": mh.MI_TYPE_F32, "f16": mh.MI_TYPE_F16, "q8": mh.MI_HIP_TYPE_Q8}[name]


class _Kv:
    """A cache handle, given back when the state goes."""

    def __init__(self, lib, *args):
        self.lib, self.h = lib, lib.kv_create(*args)

    def __del__(self):
        if getattr(self, "h", None):
            torch.cuda.synchronize()
            self.lib.mi_hip_kv_destroy(self.h)
            self.h = None


class _Rows:
    """Rows of a cache tensor in device memory, for torch.as_tensor; the cache lives as long as they do."""

    def __init__(self, kv, ptr, shape, kind):
        self.kv = kv
        self.__cuda_array_interface__ = dict(data=(ptr, False), shape=shape, typestr=kind, version=3)


def _own_rope(case, s):
    mh, lib = _lib()
    t, h, hk, d, past = (case[n] for n in ("n_tokens", "n_head", "n_head_kv", "head_dim", "n_past"))
    s["lib"], s["kv"] = lib, _Kv(lib, 1, past + t, hk, d, h, _cache_type(mh, case["cache"]))
    s["q_out"] = torch.empty_like(s["q"])
    s["args"] = mh.norm_rope_args(s["kv"].h, 0, past, d, 1e6, None, s["k"], s["v"], q=s["q"], q_out=s["q_out"],
                                  pos=s["pos"], freq=s["freq"], q_norm=s.get("q_norm"), k_norm=s.get("k_norm"), eps=1e-6)
    if case["cache"] == "q8":
        s["rows"] = [torch.empty((t, hk, d), device="cuda", dtype=torch.float16) for _ in range(2)]
    else:
        elt, kind = (4, "<f4") if case["cache"] == "f32" else (2, "<f2")
        s["rows"] = [torch.as_tensor(_Rows(s["kv"], lib.kv_view(s["kv"].h, 0, w)[0] + past * hk * d * elt, (t, hk, d),
                                           kind), device="cuda") for w in range(2)]


def _own_cache(case, s):
    mh, lib = _lib()
    t, hk, d = case["n_tokens"], case["n_head_kv"], case["head_dim"]
    s["lib"], s["kv"] = lib, _Kv(lib, 1, case["n_past"] + t, hk, d, hk, mh.MI_HIP_TYPE_Q8)
    dt = torch.float32 if case["out"] == "f32" else torch.float16
    s["rows"] = [torch.empty((case["keep"] or t, hk, d), device="cuda", dtype=dt) for _ in range(2)]


def _own_attn(case, s):
    mh, lib = _lib()
    n, t, h, hk, d = (case[x] for x in ("items", "n_tokens", "n_head", "n_head_kv", "head_dim"))
    q, out, bits = s["q"], torch.empty_like(s["q"]), s["bits"]
    s["lib"], s["out"], scale = lib, out, float(np.float32(float(d) ** -0.5))
    if case["cache"] == "q8":  # one sequence is one layer of the handle
        s["kv"] = _Kv(lib, n, case["n_past"] + t, hk, d, h, mh.MI_HIP_TYPE_Q8)
        for i in range(n):
            for w, x in enumerate((s["k_full"], s["v_full"])):
                lib.kv_write(s["kv"].h, i, w, 0, x[i], None)
        torch.cuda.synchronize()
        src = [dict(kv=s["kv"].h, layer=i) for i in range(n)]
    else:
        src = [dict(k=s["k"][i], v=s["v"][i]) for i in range(n)]
    s["items"] = (mh.AttnArgs * n)(*[mh.attn_args(q[i], out[i], h // hk, p, scale, None, **src[i])
                                     for i, p in enumerate(_pasts(case))])
    s["masks"] = mh.tree_masks([bits[i] for i in range(n)]) if bits is not None else None


def _own_logits(case, s):
    mh, s["lib"] = _lib()
    s["out"] = torch.empty_like(s["logits"])
    s["ids"] = torch.empty(case["rows"], device="cuda", dtype=torch.int32)
    s["args"] = mh.logits_args(s["logits"], s["out"], None, penalties=s["penalties"], hist=s["hist"],
                               hist_off=s["hist_off"], bias_id=s["bias_id"], bias=s["bias"], bias_off=s["bias_off"],
                               mask=s["mask"], ids=s["ids"])


def prepare(case, seed):
    kind = case["kind"]
    if kind == "attn":
        q, k, v, bits = _attn_inputs(case, seed)
        s = dict(q=q, bits=bits, n_past=torch.tensor(_pasts(case), device="cuda"))
        if case["cache"] == "q8":
            s["k"], s["v"] = _quantise(k, K_GROUP), _quantise(v, case["head_dim"])
            if own:
                s["k_full"], s["v_full"] = k, v
        else:
            dt = torch.float16 if case["cache"] == "f16" else torch.float32
            s["k"], s["v"] = k.to(dt), v.to(dt)
    else:
        s = {"norm_rope": _rope_inputs, "cache": _cache_inputs, "logits": _logits_inputs}[kind](case, seed)
    s["case"] = case
    if own:
        {"norm_rope": _own_rope, "cache": _own_cache, "attn": _own_attn, "logits": _own_logits}[kind](case, s)
        for x in ("k_full", "v_full"):
            s.pop(x, None)
    return s


# ---- one pass: the framework's calls ---------------------------------------------


def _call(s):
    lib, kind, stream = s["lib"], s["case"]["kind"], torch.cuda.current_stream().cuda_stream
    past, t = s["case"].get("n_past"), s["case"].get("n_tokens")
    if kind == "norm_rope":
        s["args"].stream = stream
        lib.check(lib.mi_hip_norm_rope_append(ctypes.byref(s["args"])))
        if s["case"]["cache"] == "q8":
            for w in range(2):
                lib.kv_read(s["kv"].h, 0, w, past, s["rows"][w], stream)
        return {"q": s["q_out"], "k": s["rows"][0], "v": s["rows"][1]}
    if kind == "cache":
        h, keep = s["kv"].h, s["keep"]
        for w, x in enumerate((s["k"], s["v"])):
            lib.kv_write(h, 0, w, past, x, stream)
        if len(keep):
            lib.kv_keep(h, past, keep, stream)
        for w in range(2):
            lib.kv_read(h, 0, w, past, s["rows"][w], stream)
        return {"k": s["rows"][0], "v": s["rows"][1]}
    if kind == "attn":
        lib.check(lib.mi_hip_attn_tree(s["items"], s["masks"], len(s["items"]), stream))
        return s["out"]
    s["args"].stream = stream
    lib.check(lib.mi_hip_logits_adjust(ctypes.byref(s["args"])))
    return {"logits": s["out"], "ids": s["ids"]}


# ---- one pass: the plain form ----------------------------------------------------


def _plain_rope(s):
    def norm(x, w):
        return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w

    # the angle is one product in 32 bits, as in the framework's other rotations
    angle = (s["pos"].float()[:, None] * torch.from_numpy(s["freq"]).cuda()).double()
    c, si = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotate(x):
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * si, a * si + b * c), -1)

    q, k, v = rotate(norm(s["q"], s.get("q_norm"))), rotate(norm(s["k"], s.get("k_norm"))), s["v"]
    if s["case"]["cache"] == "q8":
        k, v = _values(*_quantise(k, K_GROUP)), _values(*_quantise(v, v.shape[-1]))
    dt = torch.float32 if s["case"]["cache"] == "f32" else torch.float16
    return {"q": q, "k": k.to(dt), "v": v.to(dt)}


def _plain_cache(s):
    k, v = s["k"], s["v"]
    kq, vq = _quantise(k, K_GROUP), _quantise(v, v.shape[-1])
    if len(s["keep"]):
        at = torch.from_numpy(s["keep"].astype(np.int64)).cuda()
        kq, vq = [x[at] for x in kq], [x[at] for x in vq]
    dt = torch.float32 if s["case"]["out"] == "f32" else torch.float16
    return {"k": _values(*kq).to(dt), "v": _values(*vq).to(dt)}


def _visible(n_past, bits, t, n_ctx):
    """(items, t, n_ctx): which keys each query sees."""
    draft = torch.arange(n_ctx, device="cuda")[None, :] - n_past[:, None]
    if bits is None:
        return draft[:, None, :] <= torch.arange(t, device="cuda")[None, :, None]
    at = draft.clamp(0, t - 1)[:, None, :].expand(-1, t, -1)
    bit = bits.gather(2, at >> 6) >> (at & 63) & 1
    return (draft < 0)[:, None, :] | ((draft < t)[:, None, :] & (bit != 0))


def _plain_attn(s):
    q, k, v = s["q"], s["k"], s["v"]
    if s["case"]["cache"] == "q8":
        k, v = _values(*k), _values(*v)
    n, t, h, d = q.shape
    hk, n_ctx = k.shape[2], k.shape[1]
    qr = q.view(n, t, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    scores = torch.matmul(qr, k.float().permute(0, 2, 3, 1)) * float(np.float32(float(d) ** -0.5))
    seen = _visible(s["n_past"], s["bits"], t, n_ctx)
    scores = scores.view(n, hk, h // hk, t, n_ctx).masked_fill(~seen[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    o = torch.matmul(p.view(n, hk, -1, n_ctx), v.float().permute(0, 2, 1, 3)) / p.view(n, hk, -1, n_ctx).sum(-1, keepdim=True)
    return o.view(n, hk, h // hk, t, d).permute(0, 3, 1, 2, 4).reshape(n, t, h, d)


def _plain_logits(s):
    x = s["logits"]
    rows, vocab = x.shape
    row = torch.arange(rows, device="cuda")

    def rows_of(off, n):
        return torch.repeat_interleave(row, (off[1:] - off[:-1]).long(), output_size=n)

    count = torch.zeros(rows * vocab, device="cuda")
    h = s["hist"].long()
    count.index_add_(0, rows_of(s["hist_off"], len(h)) * vocab + h, torch.ones(len(h), device="cuda"))
    count = count.view(rows, vocab)
    rep, freq, presence = (s["penalties"][:, i:i + 1] for i in range(3))
    y = torch.where(x > 0, x / rep, x * rep)
    y = torch.where(count > 0, y - (count * freq + presence), x)
    b = s["bias_id"].long()
    bias = torch.zeros(rows * vocab, device="cuda")
    bias.index_add_(0, rows_of(s["bias_off"], len(b)) * vocab + b, s["bias"])
    y = y + bias.view(rows, vocab)
    if s["mask"] is not None:
        at = torch.arange(vocab, device="cuda")
        y = y.masked_fill((s["mask"][:, at >> 5] >> (at & 31) & 1) == 0, -math.inf)
    best = y.amax(-1, keepdim=True)  # the lowest index of the maximum
    ids = torch.where(y == best, torch.arange(vocab, device="cuda", dtype=torch.int32), vocab).amin(-1)
    return {"logits": y, "ids": ids.to(torch.int32)}


def run(state):
    if own:
        return _call(state)
    return {"norm_rope": _plain_rope, "cache": _plain_cache, "attn": _plain_attn,
            "logits": _plain_logits}[state["case"]["kind"]](state)


# ---- what a pass cannot do without, and its results -------------------------------


def work(case):
    kind = case["kind"]
    if kind == "logits":
        n = case["rows"] * case["vocab"]
        return {"bytes": 8 * n + (n // 8 if case["grammar"] else 0) + case["rows"] * (4 * case["history"] + 8 * case["biases"]),
                "flops": n}
    t, hk, d = case["n_tokens"], case["n_head_kv"], case["head_dim"]
    q8 = 2 + 2 / K_GROUP + 2 / d  # bytes of one dim of K and of V together
    if kind == "cache":
        rows = case["keep"] or t
        read = rows * hk * d * 2 * (4 if case["out"] == "f32" else 2)
        return {"bytes": rows * hk * d * (8 + 2 * q8) + read, "flops": 4 * rows * hk * d}
    h = case["n_head"]
    per = {"f32": 8, "f16": 4, "q8": q8}[case["cache"]]
    if kind == "norm_rope":
        out = per * (2 if case["cache"] == "q8" else 1) + (4 if case["cache"] == "q8" else 0)
        return {"bytes": t * d * (8 * h + hk * (8 + out)), "flops": 10 * t * d * (h + hk)}
    pasts = _pasts(case)
    keys = sum(pasts) + len(pasts) * t
    pairs = sum(t * p + (t if case["tree"] else t * (t + 1) // 2) for p in pasts)
    return {"bytes": keys * hk * d * per + len(pasts) * t * h * d * 8, "flops": 4 * h * d * pairs}


def _exact_scale(amax):
    a = amax / 127.0
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -14))) - 10.0)
    return torch.ceil(a / step) * step


def _exact_q8(x, group):
    """The values that the 8-bit form of x stands for."""
    x = x.double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], group):
        g = x[..., at:at + group]
        d = _exact_scale(g.abs().max(-1, keepdim=True).values)
        out[..., at:at + group] = torch.where(d > 0, torch.round(g / d.clamp_min(2.0 ** -24)) * d, 0.0 * d)
    return out


def _exact_rope(case, seed):
    s = _rope_inputs(case, seed)
    half = case["head_dim"] // 2
    theta = s["pos"].float()[:, None] * torch.as_tensor(s["freq"], device="cuda")  # one 32-bit product: the definition
    turn = torch.polar(torch.ones_like(theta, dtype=torch.float64), theta.double())[:, None]

    def both(x, w):
        x = x.double()
        if w is not None:
            x = w.double() * x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6)
        y = torch.complex(x[..., :half], x[..., half:]) * turn
        return torch.cat((y.real, y.imag), -1)

    k, v = both(s["k"], s.get("k_norm")), s["v"].double()
    if case["cache"] == "q8":
        k, v = _exact_q8(k, K_GROUP), _exact_q8(v, case["head_dim"])
    return {"q": both(s["q"], s.get("q_norm")), "k": k, "v": v}


def _exact_attn(case, seed):
    q, k, v, bits = _attn_inputs(case, seed)
    if case["cache"] == "q8":
        k, v = _exact_q8(k, K_GROUP), _exact_q8(v, case["head_dim"])
    elif case["cache"] == "f16":
        k, v = k.half(), v.half()
    t, rep = case["n_tokens"], case["n_head"] // case["n_head_kv"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    scale = float(np.float32(float(case["head_dim"]) ** -0.5))
    for i, past in enumerate(_pasts(case)):
        hidden = torch.ones((t, past + t), dtype=torch.bool, device="cuda")
        hidden[:, :past] = False
        if bits is None:
            hidden[:, past:] = torch.ones((t, t), device="cuda").triu(1) != 0
        else:
            for j in range(t):
                hidden[:, past + j] = (bits[i, :, j // 64] >> (j % 64) & 1) == 0
        for h in range(case["n_head"]):
            w = (q[i, :, h].double() @ k[i, :past + t, h // rep].double().t()) * scale
            out[i, :, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[i, :past + t, h // rep].double()
    return out


def _exact_logits(case, seed):
    s = _logits_inputs(case, seed)
    x = s["logits"].double()
    hist, h_at = s["hist"].cpu().numpy(), s["hist_off"].cpu().numpy()
    b_id, b_at, bias = s["bias_id"].cpu().numpy(), s["bias_off"].cpu().numpy(), s["bias"].double()
    for r in range(case["rows"]):
        ids, n = np.unique(hist[h_at[r]:h_at[r + 1]], return_counts=True)
        at, n = torch.from_numpy(ids.astype(np.int64)).cuda(), torch.from_numpy(n).cuda().double()
        rep, freq, presence = s["penalties"][r].double()
        was = x[r, at]
        x[r, at] = torch.where(was > 0, was / rep, was * rep) - n * freq - presence
        x[r, torch.from_numpy(b_id[b_at[r]:b_at[r + 1]].astype(np.int64)).cuda()] += bias[b_at[r]:b_at[r + 1]]
    if s["mask"] is not None:
        bits = np.unpackbits(s["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :case["vocab"]]
        x[torch.from_numpy(bits == 0).cuda()] = -math.inf
    return {"logits": x, "ids": None}


def exact(case, seed):
    if case["kind"] == "cache":
        s = _cache_inputs(case, seed)
        at = torch.from_numpy(s["keep"].astype(np.int64)).cuda() if case["keep"] else slice(None)
        return {"k": _exact_q8(s["k"], K_GROUP)[at], "v": _exact_q8(s["v"], case["head_dim"])[at]}
    return {"norm_rope": _exact_rope, "attn": _exact_attn, "logits": _exact_logits}[case["kind"]](case, seed)
