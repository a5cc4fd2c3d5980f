"""The operators of a serving step of many requests over a paged cache, as cases to be timed.

A program that serves many requests at once keeps their K and V in pages of a
common pool, and makes these calls each step (include/mi_hip_attn.h):

  tables   mi_hip_page_tables: from the requests' lengths, on the GPU: pages taken
           from and given back to the pool, the block tables, each token's cache
           row and position;
  append   mi_hip_paged_append: the norms of queries and keys per head (models
           that have them), the rotation by positions of one or several axes
           (text, image patches, video), and the append of K and V to those rows
           of an F32, F16 or 8-bit cache;
  attn     mi_hip_attn_paged: attention of each request's new tokens (one, a few
           drafted ones, a prompt's chunk) over its pages;
  verify   mi_hip_verify_draft: which drafted tokens the target's probabilities
           accept, and the token after them, from given random numbers.

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


def _tables(n_seq, cached, chunk, page, tight=False):
    return dict(kind="tables", n_seq=n_seq, cached=cached, chunk=chunk, page=page, tight=tight)


def _append(n_tokens, axes, turns, cache, page, shape, norm=False, n_dims=0):
    return dict(kind="append", n_tokens=n_tokens, axes=axes, turns=turns, cache=cache, page=page, norm=norm,
                n_dims=n_dims or shape["head_dim"], **shape)


def _attn(n_seq, past, new, n_chunk, chunk_past, chunk, cache, page, shape):
    return dict(kind="attn", n_seq=n_seq, past=past, new=new, n_chunk=n_chunk, chunk_past=chunk_past, chunk=chunk,
                cache=cache, page=page, **shape)


def _verify(n_seq, nodes, vocab, draft, tree, greedy=False):
    return dict(kind="verify", n_seq=n_seq, nodes=nodes, vocab=vocab, draft=draft, tree=tree, greedy=greedy)


def listed():
    def named(name, c):
        return dict(c, name=name)
    return [
        # eight chats, a token each: latency
        named("tables_8", _tables(8, 600, 1, 16)),
        # a server's batch: chats, drafted tokens turned down, requests that end, prompts' chunks
        named("tables_1024", _tables(1024, 4096, 500, 64)),
        # one generated token of eight chats, F32 cache: latency
        named("append_8_f32", _append(8, 1, False, "f32", 16, QWEN05B)),
        # an image's patches by time, height and width, axes in sections, 8-bit cache
        named("append_1225_image_q8", _append(1225, 3, False, "q8", 32, QWEN7B)),
        # a step's prompts and chats with frames of a video, axes in turn, norms, F16 cache
        named("append_8192_video_f16", _append(8192, 3, True, "f16", 64, QWEN7B, norm=True)),
        # one token early in one chat, F16 cache: latency
        named("attn_1x500_f16", _attn(1, 499, 1, 0, 0, 0, "f16", 16, QWEN05B)),
        # a token of each of 64 long chats, 8-bit cache
        named("attn_64x8192_q8", _attn(64, 8191, 1, 0, 0, 0, "q8", 32, QWEN7B)),
        # five drafted tokens and the one before them of 32 chats, F32 cache
        named("attn_32x6x3000_f32", _attn(32, 2994, 6, 0, 0, 0, "f32", 16, QWEN05B)),
        # a prompt's chunk among 31 chats, F16 cache
        named("attn_mixed_1000_f16", _attn(31, 4000, 1, 1, 1337, 1000, "f16", 64, QWEN7B)),
        # a chunk far into a long prompt, F16 cache
        named("attn_chunk_2048x8048_f16", _attn(0, 0, 0, 1, 6000, 2048, "f16", 128, QWEN7B)),
        # one chat's drafted tokens taken as certain (n-gram lookup): latency
        named("verify_1x6", _verify(1, 6, VOCAB, False, False)),
        # a batch's chains of tokens drawn from a draft model
        named("verify_64x6_draft", _verify(64, 6, VOCAB, True, False)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "append", "attn", "attn", "attn", "verify", "verify"])
    page = rng.choice([16, 32, 64, 128, 256])
    shape = rng.choice([QWEN05B, QWEN7B])
    cache = rng.choice(["f32", "f16", "q8"])
    if kind == "tables":
        return _tables(_log(rng, 1, 1024), _log(rng, 16, 8192), _log(rng, 1, 1000), page, rng.random() < 0.3)
    if kind == "append":
        dims = shape["head_dim"] if rng.random() < 0.8 else shape["head_dim"] // 2
        return _append(_log(rng, 1, 8192), rng.randint(1, 4), rng.random() < 0.5, cache, page, shape,
                       norm=rng.random() < 0.5, n_dims=dims)
    if kind == "verify":
        draft = rng.random() < 0.5
        nodes = rng.randint(1, 8) if draft or rng.random() < 0.5 else rng.randint(9, 40)
        n_seq = max(1, min(_log(rng, 1, 64), 384 // nodes))
        return _verify(n_seq, nodes, rng.choice([VOCAB, _log(rng, 1000, VOCAB)]), draft, not draft and rng.random() < 0.7,
                       rng.random() < 0.2)
    n_chunk = rng.choice([0, 0, 1, 1, 2])
    chunk = _log(rng, 8, 2048) if n_chunk else 0
    chunk_past = rng.choice([0, _log(rng, 1, 8192)]) if n_chunk else 0
    chunk = max(1, min(chunk, (1 << 23) // (n_chunk * (chunk_past + 1024)))) if n_chunk else 0
    n_seq = _log(rng, 1, 64) if not n_chunk or rng.random() < 0.6 else 0
    new = rng.choice([1, 1, rng.randint(2, 12)]) if n_seq else 0
    past = _log(rng, 1, 16384) if n_seq else 0
    # at most 400 MB of keys and values
    per = shape["n_head_kv"] * shape["head_dim"] * {"f32": 8, "f16": 4, "q8": 2.2}[cache]
    if n_seq:
        n_seq = max(1, min(n_seq, int(400e6 / per) // (past + new)))
    return _attn(n_seq, past, new, n_chunk, chunk_past, chunk, cache, page, shape)


# ---- inputs -------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


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


def _requests(case, seed):
    """(cached, new, held pages) of each request: chats that generate a token, chats whose drafted
    tokens were turned down (they hold pages they need no more), new and running prompts' chunks,
    and requests that end. Another seed has them in another order."""
    rng = np.random.RandomState(case["n_seq"] * 1000 + case["cached"])
    n, page = case["n_seq"], case["page"]
    cached = np.maximum(1, (case["cached"] * rng.uniform(0.2, 1.0, n)).astype(np.int64))
    new = np.ones(n, np.int64)
    held = -(-cached // page)
    role = rng.randint(0, 16, n) if n > 8 else np.full(n, 15)
    new[role == 0] = rng.randint(1, case["chunk"] + 1, n)[role == 0]
    cached[role == 1], held[role == 1] = 0, 0
    new[role == 1] = rng.randint(1, case["chunk"] + 1, n)[role == 1]
    held[role == 2] += rng.randint(0, 3, n)[role == 2]
    new[role == 2] = 6
    cached[role == 3], new[role == 3] = 0, 0
    order = np.random.RandomState(seed & 0x7FFFFFFF).permutation(n)
    return cached[order], new[order], held[order]


def _tables_inputs(case, seed):
    cached, new, held = _requests(case, seed)
    rng = np.random.RandomState((seed + 1) & 0x7FFFFFFF)
    n, page = case["n_seq"], case["page"]
    need = -(-(cached + new) // page)
    width = int(max(need.max(), held.max())) + 3
    taken = int(np.maximum(need - held, 0).sum())
    free = taken // 2 if case["tight"] else taken + 5
    n_pages = int(held.sum()) + free + 7  # (seven are with someone else)
    ids = rng.permutation(n_pages)
    table = np.full((n, width), -1, np.int64)
    table[np.arange(width)[None, :] < held[:, None]] = ids[:held.sum()]
    head = int(rng.randint(0, n_pages))
    ring = np.full(n_pages, -1, np.int64)
    ring[(head + np.arange(free)) % n_pages] = ids[held.sum():held.sum() + free]
    total = int(new.sum())
    s = dict(cached=_ints(cached), new=_ints(new), held=_ints(held), table=_ints(table), ring=_ints(ring),
             ring_at=_ints([head, head + free]), n_tokens=total + 3)  # a batch is padded to a size of its own
    return s


def _axis_of(case):
    """The axis of each pair of dims: sections one after the other (a quarter for the first axis,
    the rest alike), or the axes in turn."""
    pairs, axes = case["n_dims"] // 2, case["axes"]
    if case["turns"] or axes == 1:
        return [i % axes for i in range(pairs)]
    first = pairs // 4
    return [0 if i < first else 1 + (i - first) * (axes - 1) // (pairs - first) for i in range(pairs)]


def _append_inputs(case, seed):
    g = _gen(seed)
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    t, h, hk, d, page = case["n_tokens"], case["n_head"], case["n_head_kv"], case["head_dim"], case["page"]
    s = dict(q=torch.randn((t, h, d), device="cuda", generator=g) * 2.0, k=_keys((t, hk, d), g),
             v=torch.randn((t, hk, d), device="cuda", generator=g))
    if case["norm"]:
        s["q_norm"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
        s["k_norm"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)
    n = case["n_dims"]
    s["freq"] = (1e6 ** (-np.arange(0, n, 2, dtype=np.float64) / n)).astype(np.float32)
    # patches of frames 35 wide, row by row, after some text; one axis: the tokens in order
    at, base = np.arange(t), int(rng.randint(0, 4096))
    pos = np.stack([at] if case["axes"] == 1 else [at // 1225, at % 1225 // 35, at % 35, at // 35][:case["axes"]])
    s["pos"] = _ints(base + pos)
    # the rows of a pool's pages in any order; the last two tokens of a longer batch are padding
    s["n_pages"] = -(-t // page)
    slots = rng.permutation(s["n_pages"])[at // page] * page + at % page
    if t > 8:
        slots[-2:] = -1
    s["slots"] = _ints(slots)
    return s


def _lengths(case):
    """(cached before, new) of each request: ragged, the first of a kind the longest."""
    n, m = case["n_seq"], case["n_chunk"]
    chats = [(case["past"] - i * case["past"] // (3 * n), case["new"]) for i in range(n)]
    chunks = [(case["chunk_past"] - i * case["chunk_past"] // (3 * m), case["chunk"]) for i in range(m)]
    return chunks + chats


def _attn_inputs(case, seed):
    g = _gen(seed)
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    page, hk, d = case["page"], case["n_head_kv"], case["head_dim"]
    lens = _lengths(case)
    pages = [-(-(p + n) // page) for p, n in lens]
    n_pages = sum(pages) + 3
    ids = rng.permutation(n_pages)
    table = np.full((len(lens), max(pages) + 1), -1, np.int64)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = ids[at:at + n]
        at += n
    t = sum(n for _, n in lens)
    shape = (n_pages * page, hk, d)
    return dict(q=torch.randn((t, case["n_head"], d), device="cuda", generator=g), table=_ints(table), n_pages=n_pages,
                q_off=_ints(np.concatenate([[0], np.cumsum([n for _, n in lens])])), n_kv=_ints([p + n for p, n in lens]),
                k=_keys(shape, g) * 0.5, v=torch.randn(shape, device="cuda", generator=g))


def _verify_inputs(case, seed):
    g = _gen(seed)
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    n, vocab = case["n_seq"], case["vocab"]
    # trees and certain tokens come in numbers of their own for each request
    count = np.full(n, case["nodes"]) if case["draft"] else rng.randint((case["nodes"] + 1) // 2, case["nodes"] + 1, n)
    off = np.concatenate([[0], np.cumsum(count)])
    rows = int(off[-1])
    logits = torch.randn((rows, vocab), device="cuda", generator=g) * 3.0
    temperature = np.where(rng.rand(n) < 0.5, 1.0, 0.7).astype(np.float32)
    if case["greedy"]:
        temperature[rng.rand(n) < 0.7] = 0.0
    s = dict(logits=logits, temperature=torch.from_numpy(temperature).cuda(), off=_ints(off),
             u=torch.rand(rows, device="cuda", generator=g), parent=None, draft=None)
    parent = np.maximum(np.concatenate([np.arange(c) for c in count]) - 1, 0)
    if case["tree"]:
        parent = np.concatenate([[0] + [rng.randint(max(0, i - 4), i) for i in range(1, c)] for c in count])
        s["parent"] = _ints(parent)
    row = torch.from_numpy(parent + np.repeat(off[:-1], count)).cuda()  # each node's parent's row
    if case["draft"]:
        # a draft model that is close to the target
        guess = logits[row] + 1.5 * torch.randn((rows, vocab), device="cuda", generator=g)
        s["draft"] = torch.softmax(guess, -1)
        token = torch.multinomial(s["draft"], 1, generator=g)[:, 0]
    else:
        # likely tokens: the siblings of a tree take the parent's best in turn
        rank = np.zeros(rows, np.int64)
        seen = {}
        for i, r in enumerate(row.cpu().tolist()):
            rank[i] = seen[r] = seen.get(r, -1) + 1
        best = torch.topk(logits, min(vocab, int(rank.max()) + 1), -1).indices
        token = best[row, torch.from_numpy(rank).cuda()]
    s["token"] = token.to(torch.int32)
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
        self.lib, self.h = lib, lib.kv_create_paged(*args)

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


def _own_tables(case, s):
    mh, s["lib"] = _lib()
    n, t = case["n_seq"], s["n_tokens"]
    s["out"] = {k: torch.empty(m, dtype=torch.int32, device="cuda")
                for k, m in (("held", n), ("ring_at", 2), ("n_kv", n), ("q_off", n + 1), ("slots", t), ("pos", t), ("seq", t),
                             ("refused", 1))}
    o = s["out"]
    s["args"] = mh.page_tables_args(case["page"], s["cached"], s["new"], s["held"], o["held"], s["table"], s["ring"],
                                    s["ring_at"], o["ring_at"], o["n_kv"], o["q_off"], o["slots"], None, pos=o["pos"],
                                    seq=o["seq"], n_refused=o["refused"])
    o["table"], o["ring"] = s["table"], s["ring"]


def _own_append(case, s):
    mh, lib = _lib()
    h, hk, d, page = (case[n] for n in ("n_head", "n_head_kv", "head_dim", "page"))
    rows = s["n_pages"] * page
    s["lib"], s["kv"] = lib, _Kv(lib, 1, s["n_pages"], page, hk, d, h, _cache_type(mh, case["cache"]))
    s["q_out"] = torch.empty_like(s["q"])
    s["args"] = mh.paged_append_args(s["kv"].h, 0, case["n_dims"], 1e6, None, s["k"], s["v"], s["slots"], s["pos"], q=s["q"],
                                     q_out=s["q_out"], axis=_axis_of(case), freq=s["freq"], q_norm=s.get("q_norm"),
                                     k_norm=s.get("k_norm"), eps=1e-6)
    if case["cache"] == "q8":
        s["rows"] = [torch.empty((rows, hk, d), device="cuda", dtype=torch.float16) for _ in range(2)]
    else:
        kind = "<f4" if case["cache"] == "f32" else "<f2"
        s["rows"] = [torch.as_tensor(_Rows(s["kv"], lib.kv_view(s["kv"].h, 0, w)[0], (rows, hk, d), kind), device="cuda")
                     for w in range(2)]


def _own_attn(case, s):
    mh, lib = _lib()
    h, hk, d, page = (case[n] for n in ("n_head", "n_head_kv", "head_dim", "page"))
    s["lib"], s["kv"] = lib, _Kv(lib, 1, s["n_pages"], page, hk, d, h, _cache_type(mh, case["cache"]))
    for w, x in enumerate((s["k_full"], s["v_full"])):
        lib.kv_write(s["kv"].h, 0, w, 0, x, None)
    torch.cuda.synchronize()
    s["out"] = torch.empty_like(s["q"])
    s["args"] = mh.paged_attn_args(s["kv"].h, 0, s["q"], s["out"], s["q_off"], s["n_kv"], s["table"],
                                   float(np.float32(float(d) ** -0.5)), None, max_new=max(n for _, n in _lengths(case)))


def _own_verify(case, s):
    mh, s["lib"] = _lib()
    n, most = case["n_seq"], case["nodes"]
    s["out"] = dict(n_path=torch.empty(n, dtype=torch.int32, device="cuda"),
                    path=torch.empty((n, most), dtype=torch.int32, device="cuda"),
                    tokens=torch.empty((n, most), dtype=torch.int32, device="cuda"))
    s["args"] = mh.verify_args(s["logits"], s["off"], s["token"], s["u"], s["out"]["n_path"], s["out"]["path"],
                               s["out"]["tokens"], None, parent=s["parent"], draft=s["draft"], temperature=s["temperature"])


def prepare(case, seed):
    kind = case["kind"]
    s = {"tables": _tables_inputs, "append": _append_inputs, "attn": _attn_inputs, "verify": _verify_inputs}[kind](case, seed)
    if kind == "attn":
        if own:
            s["k_full"], s["v_full"] = s["k"], s["v"]
        if case["cache"] == "q8":
            s["k"], s["v"] = _quantise(s["k"], K_GROUP), _quantise(s["v"], case["head_dim"])
        elif case["cache"] == "f16":
            s["k"], s["v"] = s["k"].half(), s["v"].half()
        if own:  # the cache has them
            del s["k"], s["v"]
    if kind == "append" and not own:
        dt = torch.float32 if case["cache"] == "f32" else torch.float16
        shape = (s["n_pages"] * case["page"], case["n_head_kv"], case["head_dim"])
        s["rows"] = [torch.zeros(shape, device="cuda", dtype=dt) for _ in range(2)]
    s["case"] = case
    if own:
        {"tables": _own_tables, "append": _own_append, "attn": _own_attn, "verify": _own_verify}[kind](case, s)
        for x in ("k_full", "v_full"):
            s.pop(x, None)
    return s


# ---- one pass: the framework's calls ---------------------------------------------


def _call(s):
    lib, kind = s["lib"], s["case"]["kind"]
    s["args"].stream = torch.cuda.current_stream().cuda_stream
    args = ctypes.byref(s["args"])
    if kind == "tables":
        lib.check(lib.mi_hip_page_tables(args))
        return s["out"]
    if kind == "append":
        lib.check(lib.mi_hip_paged_append(args))
        if s["case"]["cache"] == "q8":
            for w in range(2):
                lib.kv_read(s["kv"].h, 0, w, 0, s["rows"][w], s["args"].stream)
        return {"q": s["q_out"], "k": s["rows"][0], "v": s["rows"][1]}
    if kind == "attn":
        lib.check(lib.mi_hip_attn_paged(args))
        return s["out"]
    lib.check(lib.mi_hip_verify_draft(args))
    return s["out"]


# ---- one pass: the plain form ----------------------------------------------------


def _plain_tables(s):
    page, t, width = s["case"]["page"], s["n_tokens"], s["table"].shape[1]
    cached, new, held = s["cached"].long(), s["new"].long(), s["held"].long()
    head, tail = s["ring_at"].long()
    n_pages = len(s["ring"])
    need = (cached + new + page - 1) // page
    fits = need <= width
    take = torch.where(fits, (need - held).clamp_min(0), 0)
    end = take.cumsum(0)
    refused = ~fits | ((take > 0) & (end > tail - head))
    q_end = new.cumsum(0)
    take = torch.where(refused, 0, take)
    give = torch.where(refused, 0, (held - need).clamp_min(0))
    at = torch.arange(width, device="cuda")[None, :]
    first = (end - take)[:, None] - held[:, None]
    new_page = (at >= held[:, None]) & (at < (held + take)[:, None])
    old = s["table"]
    table = torch.where(new_page, s["ring"][(head + first + at) % n_pages], old)
    gone = (at >= (held - give)[:, None]) & (at < held[:, None])
    to = (tail + (give.cumsum(0) - give)[:, None] + at - (held - give)[:, None]) % n_pages
    # (one ring entry more takes what is not given back)
    ring = torch.cat((s["ring"], s["ring"].new_zeros(1)))
    ring.scatter_(0, torch.where(gone, to, n_pages).flatten(), old.flatten())
    tok = torch.arange(t, device="cuda")
    n = len(new)
    seq = (tok[:, None] >= q_end[None, :]).sum(1)
    real = seq < n
    sq = seq.clamp_max(n - 1)
    pos = torch.where(real, cached[sq] + tok - (q_end - new)[sq], 0)
    entry = table[sq, (pos // page).clamp_max(width - 1)].long()
    slots = torch.where(real & ~refused[sq], entry * page + pos % page, -1)
    i32 = torch.int32
    head, tail = head + take.sum(), tail + give.sum()
    laps = head // n_pages * n_pages
    return {"held": (held + take - give).to(i32), "ring_at": torch.stack((head - laps, tail - laps)).to(i32),
            "n_kv": torch.where(refused, 0, cached + new).to(i32),
            "q_off": torch.cat((q_end.new_zeros(1), q_end)).to(i32), "slots": slots.to(i32), "pos": pos.to(i32),
            "seq": torch.where(real, seq, -1).to(i32), "refused": refused.sum()[None].to(i32), "table": table,
            "ring": ring[:n_pages]}


def _plain_append(s):
    case = s["case"]
    n = case["n_dims"]

    def norm(x, w):
        return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w

    # the angle is one product in 32 bits, as in the framework's other rotations
    pos = s["pos"].float()[torch.tensor(_axis_of(case), device="cuda")].t()
    angle = (pos * torch.from_numpy(s["freq"]).cuda()).double()
    c, si = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotate(x):
        a, b = x[..., :n].chunk(2, -1)
        return torch.cat((a * c - b * si, a * si + b * c, x[..., n:]), -1)

    q, k, v = rotate(norm(s["q"], s.get("q_norm"))), rotate(norm(s["k"], s.get("k_norm"))), s["v"]
    if case["cache"] == "q8":
        k, v = _values(*_quantise(k, K_GROUP)), _values(*_quantise(v, v.shape[-1]))
    keep = s["slots"] >= 0
    at = s["slots"][keep].long()
    for rows, x in zip(s["rows"], (k, v)):
        rows[at] = x[keep].to(rows.dtype)
    return {"q": q, "k": s["rows"][0], "v": s["rows"][1]}


def _plain_attn(s):
    case = s["case"]
    q, page, hk, d = s["q"], case["page"], case["n_head_kv"], case["head_dim"]
    h = case["n_head"]
    out = torch.empty_like(q)
    scale = float(np.float32(float(d) ** -0.5))
    lens = _lengths(case)
    # requests with as many new tokens go together, shorter ones padded
    i = row = 0
    while i < len(lens):
        j, t = i, lens[i][1]
        while j < len(lens) and lens[j][1] == t:
            j += 1
        n, n_kv = j - i, s["n_kv"][i:j]
        most = max(p for p, _ in lens[i:j]) + t
        key = torch.arange(most, device="cuda")
        at = s["table"][i:j, key // page].clamp_min(0).long() * page + key % page
        if case["cache"] == "q8":
            k, v = (_values(x[0][at], x[1][at]) for x in (s["k"], s["v"]))
        else:
            k, v = s["k"][at].float(), s["v"][at].float()
        qr = q[row:row + n * t].view(n, t, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
        scores = torch.matmul(qr, k.permute(0, 2, 3, 1).contiguous()) * scale
        seen = key[None, None, :] <= (n_kv - t)[:, None, None] + torch.arange(t, device="cuda")[None, :, None]
        scores = scores.view(n, hk, h // hk, t, most).masked_fill(~seen[:, None, None], -math.inf)
        p = (scores - scores.amax(-1, keepdim=True)).exp().view(n, hk, -1, most)
        o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous()) / p.sum(-1, keepdim=True)
        out[row:row + n * t] = o.view(n, hk, h // hk, t, d).permute(0, 3, 1, 2, 4).reshape(n * t, h, d)
        i, row = j, row + n * t
    return out


def _plain_verify(s):
    # in 64 bits: the outputs are whole numbers
    case = s["case"]
    most, vocab = case["nodes"], case["vocab"]
    off = s["off"].long()
    first, count = off[:-1], off[1:] - off[:-1]
    n = len(first)
    seq = torch.arange(n, device="cuda")
    t = s["temperature"].double()[torch.repeat_interleave(seq, count, output_size=len(s["logits"]))][:, None]
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    w = torch.exp(x / torch.where(t > 0, t, 1.0))
    best = torch.where(x == 0, torch.arange(vocab, device="cuda"), vocab).amin(-1, keepdim=True)
    w = torch.where(t > 0, w, (torch.arange(vocab, device="cuda") == best).double())
    p = w / w.sum(-1, keepdim=True)
    token = s["token"].long()
    u = s["u"].double()
    cur = torch.zeros_like(first)
    left = torch.ones(n, dtype=torch.float64, device="cuda")
    path = torch.full((n, most), -1, dtype=torch.int64, device="cuda")
    tokens = torch.full((n, most), -1, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    n_path = torch.ones_like(first)
    down = torch.zeros((n, most), dtype=torch.bool, device="cuda")  # children of cur that were turned down
    for c in range(1, most):
        r = (first + c).clamp_max(len(token) - 1)
        up = torch.full_like(cur, c - 1) if s["parent"] is None else s["parent"][r].long()
        child = (c < count) & (up == cur)
        again = torch.zeros_like(child)
        for e in range(1, c):
            again |= down[:, e] & (token[(first + e).clamp_max(len(token) - 1)] == token[r])
        pc = torch.where(again, 0.0, p[first + cur, token[r]])
        bar = u[r] * (left if s["draft"] is None else s["draft"][r, token[r]].double())
        yes = child & (bar < pc)
        tokens[seq, n_path - 1] = torch.where(yes, token[r], tokens[seq, n_path - 1])
        at = n_path.clamp_max(most - 1)
        path[seq, at] = torch.where(yes, c, path[seq, at])
        n_path = n_path + yes
        left = torch.where(yes, 1.0, torch.where(child, left - pc, left))
        cur = torch.where(yes, c, cur)
        down &= ~yes[:, None]
        down[:, c] = child & ~yes
    rest = p[first + cur]
    for c in range(1, most):
        r = (first + c).clamp_max(len(token) - 1)
        if s["draft"] is None:
            rest[seq, token[r]] = torch.where(down[:, c], 0.0, rest[seq, token[r]])
        else:
            rest = torch.where(down[:, c, None], (rest - s["draft"][r].double()).clamp_min(0.0), rest)
    total = rest.cumsum(-1)
    bar = u[first][:, None] * total[:, -1:]
    drawn = (total <= bar).sum(-1)
    tokens[seq, n_path - 1] = drawn
    i32 = torch.int32
    return {"n_path": n_path.to(i32), "path": path.to(i32), "tokens": tokens.to(i32)}


def run(state):
    if own:
        return _call(state)
    return {"tables": _plain_tables, "append": _plain_append, "attn": _plain_attn,
            "verify": _plain_verify}[state["case"]["kind"]](state)


# ---- what a pass cannot do without, and its results -------------------------------


def work(case):
    kind = case["kind"]
    if kind == "tables":
        cached, new, held = _requests(case, 1)
        need = -(-(cached + new) // case["page"])
        pages = int(np.abs(need - held).sum())
        blocks = int((new // case["page"] + (new > 0)).sum())  # table entries that the slots come from
        return {"bytes": 4 * (6 * case["n_seq"] + 2 * pages + blocks + 3 * int(new.sum())),
                "flops": 4 * case["n_seq"] + 3 * int(new.sum())}
    if kind == "verify":
        mean = case["nodes"] if case["draft"] else (case["nodes"] + (case["nodes"] + 1) // 2) / 2
        rows = int(case["n_seq"] * mean)
        # the logits, and the draft's row where a chain ends
        return {"bytes": 4 * case["vocab"] * (rows + (case["n_seq"] if case["draft"] else 0)), "flops": 20 * rows * case["vocab"]}
    hk, d, h = case["n_head_kv"], case["head_dim"], case["n_head"]
    per = {"f32": 8, "f16": 4, "q8": 2 + 2 / K_GROUP + 2 / d}[case["cache"]]  # one dim of K and of V together
    if kind == "append":
        t = case["n_tokens"]
        out = per * (2 if case["cache"] == "q8" else 1) + (4 if case["cache"] == "q8" else 0)
        return {"bytes": t * d * (8 * h + hk * (8 + out)), "flops": 10 * t * d * (h + hk)}
    lens = _lengths(case)
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in lens)
    return {"bytes": int(sum(p + n for p, n in lens) * hk * d * per + sum(n for _, n in lens) * h * d * 8),
            "flops": 4 * h * d * pairs}


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


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    half = case["n_dims"] // 2
    pos = torch.stack([s["pos"][a] for a in _axis_of(case)], 1)
    theta = pos.float() * torch.as_tensor(s["freq"], device="cuda")  # one 32-bit product: the definition
    turn = torch.polar(torch.ones_like(theta, dtype=torch.float64), theta.double())[:, None]

    def both(x, w):
        x = x.double()
        if w is not None:
            x = w.double() * x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6)
        y = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        return torch.cat((y.real, y.imag, x[..., 2 * half:]), -1)

    k, v = both(s["k"], s.get("k_norm")), s["v"].double()
    if case["cache"] == "q8":
        k, v = _exact_q8(k, K_GROUP), _exact_q8(v, case["head_dim"])
    rows = []
    slots = s["slots"].long()
    for x in (k, v):
        r = torch.zeros((s["n_pages"] * case["page"], case["n_head_kv"], case["head_dim"]), dtype=torch.float64, device="cuda")
        r.index_copy_(0, slots[slots >= 0], x[slots >= 0])
        rows.append(r)
    return {"q": both(s["q"], s.get("q_norm")), "k": rows[0], "v": rows[1]}


def _exact_attn(case, seed):
    s = _attn_inputs(case, seed)
    k, v, q, page = s["k"], s["v"], s["q"], case["page"]
    if case["cache"] == "q8":
        k, v = _exact_q8(k, K_GROUP), _exact_q8(v, case["head_dim"])
    elif case["cache"] == "f16":
        k, v = k.half(), v.half()
    rep = case["n_head"] // case["n_head_kv"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    scale = float(np.float32(float(case["head_dim"]) ** -0.5))
    row = 0
    for i, (past, t) in enumerate(_lengths(case)):
        pages = s["table"][i, :-(-(past + t) // page)].long()
        rows = (pages[:, None] * page + torch.arange(page, device="cuda")).flatten()[:past + t]
        hidden = torch.zeros((t, past + t), dtype=torch.bool, device="cuda")
        hidden[:, past:] = torch.ones((t, t), device="cuda").triu(1) != 0
        for h in range(case["n_head"]):
            w = (q[row:row + t, h].double() @ k[rows, h // rep].double().t()) * scale
            out[row:row + t, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[rows, h // rep].double()
        row += t
    return out


def exact(case, seed):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(case, seed)
    return None  # whole numbers
