"""Edges of the operators over a paged cache: workspaces without parts, pools whose offsets pass 32 bits,
pages shared by sequences, more sequences than arrival counters, temperatures that are no numbers."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import paged_ref
import serve_ref as ref
from test_kv8_gpu import dev, read
from test_paged_attn_gpu import KINDS, Batch
from test_verify_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("d,hkv,rep,seqs", [(64, 2, 7, [(2500, 1), (3, 2), (900, 4)]), (128, 2, 4, [(1100, 9), (700, 300), (40, 1)]),
                                            (64, 1, 16, [(1500, 40)])])
def test_caches_without_room_for_parts(hip, stream, cache, d, hkv, rep, seqs):
    """Then every sequence's keys stay in one piece. The same calls with a workspace that has parts agree."""
    rng = np.random.default_rng([d, rep])
    before = hip.alloc_stats().bytes_live
    kv = hip.kv_create_paged(2, -(-sum(n + 15 for n, _ in seqs) // 16) + 2, 16, hkv, d, hkv * rep, KINDS[cache])
    whole = hip.alloc_stats().bytes_live - before
    hip.check(hip.mi_hip_kv_destroy(kv))
    try:
        hip.check(hip.mi_hip_set_alloc_limit(before + whole - (1 << 20)))
        b = Batch(hip, rng, cache, d, hkv, rep, 16, seqs, lead=1, tail=1)
        assert hip.alloc_stats().bytes_live - before < whole - (16 << 20)
    finally:
        hip.check(hip.mi_hip_set_alloc_limit(0))
    got = b.run(stream)
    b.check(got)
    assert np.array_equal(got, b.run(stream))
    ws = hip.workspace_create(hkv, hkv * rep, d)
    b.check(b.run(stream, ws=ws))
    hip.check(hip.mi_hip_workspace_destroy(ws))
    b.close()


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("new", [3, 70])
def test_pools_beyond_32_bits(hip, stream, cache, new):
    """Pages at both sides of the 2^32th byte of K: appended, read back, attended over."""
    import torch
    rng = np.random.default_rng([new, list(KINDS).index(cache)])
    d, hkv, rep, page = 128, 4, 2, 16
    row = hkv * d * {"f32": 4, "f16": 2, "q8": 1}[cache]
    edge = (1 << 32) // row // page  # the first page beyond
    kv = hip.kv_create_paged(1, edge + 40, page, hkv, d, hkv * rep, KINDS[cache])
    n_kv = [330, 95]
    pages = [-(-n // page) for n in n_kv]
    ids = np.concatenate([edge + np.arange(12), edge - 1 - np.arange(12), [0, 1, edge + 39, (1 << 31) // row // page]])
    ids = rng.permutation(ids)[:sum(pages)]
    assert (ids >= edge).any() and (ids < edge).any()
    table = np.full((2, max(pages)), -1, np.int32)
    table[0, :pages[0]], table[1, :pages[1]] = ids[:pages[0]], ids[pages[0]:]
    slots = np.concatenate([table[i, np.arange(n) // page] * page + np.arange(n) % page for i, n in enumerate(n_kv)])
    t = len(slots)
    k, v = (rng.standard_normal((t, hkv, d)).astype(np.float32) for _ in range(2))
    a = mh.paged_append_args(kv, 0, d, 1e6, stream, dev(k), dev(v), dev(slots.astype(np.int32)),
                             torch.zeros(t, dtype=torch.int32, device="cuda"))
    hip.check(hip.mi_hip_paged_append(ctypes.byref(a)))  # (position 0: no rotation)
    torch.cuda.synchronize()
    if cache == "f16":
        k, v = (x.astype(np.float16).astype(np.float32) for x in (k, v))
    elif cache == "q8":
        k, v = ref.q8(k, 0), ref.q8(v, 1)
    for e, i in ((0, 0), (1, n_kv[0])):
        for which, x in ((0, k), (1, v)):
            got = read(hip, kv, 0, which, int(table[e, 0]) * page, page, hkv, d, stream)
            assert np.array_equal(got, x[i:i + page])
    q = rng.standard_normal((2 * new, hkv * rep, d)).astype(np.float32)
    out = torch.full(q.shape, 7.5, device="cuda")
    scale = float(np.float32(d ** -0.5))
    a = mh.paged_attn_args(kv, 0, dev(q), out, dev(np.array([0, new, 2 * new], np.int32)), dev(np.array(n_kv, np.int32)), dev(table),
                           scale, stream)
    hip.check(hip.mi_hip_attn_paged(ctypes.byref(a)))
    torch.cuda.synchronize()
    at = 0
    for i, n in enumerate(n_kv):
        x, kk, vv = q[i * new:(i + 1) * new], k[at:at + n], v[at:at + n]
        seen = np.arange(n)[None, :] <= (n - new + np.arange(new))[:, None]
        err = np.abs(out.cpu().numpy()[i * new:(i + 1) * new] - ref.attention(x, kk, vv, seen, scale)).max()
        assert err <= ref.attention_tolerance(x, kk, vv, seen, scale)
        at += n
    hip.check(hip.mi_hip_kv_destroy(kv))


@pytest.mark.parametrize("cache", list(KINDS))
def test_pages_shared_by_sequences(hip, stream, cache):
    """A prompt's pages stand in several tables, one of them twice in a row of its own."""
    b = Batch(hip, np.random.default_rng(3), cache, 64, 2, 7, 16, [(160, 2), (200, 1), (130, 40), (64, 3)])
    b.table[1, :8] = b.table[0, :8]
    b.table[2, :8] = b.table[0, :8]
    b.table[3, 1] = b.table[3, 0]
    b.dtable.copy_(dev(b.table))
    b.check(b.run(stream))
    b.close()


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("d,hkv,rep,seqs", [
    (64, 2, 7, [(1500 - 7 * i, 1) for i in range(64)]),               # shares a little larger, no workgroup with two units
    (64, 2, 7, [(1500 - 11 * i, 6) for i in range(32)]),              # the same, more than 16 rows
    (128, 4, 7, [(100, 100)]),                                        # row tiles of few keys, each whole
    (128, 4, 7, [(250, 250)]),                                        # and of a few more, in parts
    (128, 2, 7, [(1000 + i, 1) for i in range(8)] + [(300, 300)]),    # two short lines
    (64, 2, 7, [(700, 1), (40, 1), (3, 1), (520, 30), (64, 64)]),
    (64, 1, 7, [(40 + i % 90, 1) for i in range(300)] + [(20 + i % 50, 20) for i in range(300)]),  # more units than workgroups
])
def test_shares(hip, stream, cache, d, hkv, rep, seqs):
    """Lengths on both sides of the rules by which units are cut into shares."""
    b = Batch(hip, np.random.default_rng([d, len(seqs)]), cache, d, hkv, rep, 16, seqs, lead=1, tail=2)
    got = b.run(stream)
    b.check(got)
    assert np.array_equal(got, b.run(stream))
    b.check(b.run(stream, max_new=max(n for _, n in seqs)), "max_new")
    b.close()


def softmax_rows(rng, rows, vocab):
    x = rng.standard_normal((rows, vocab))
    e = np.exp(x - x.max(1, keepdims=True))
    return (e / e.sum(1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("drafted", [False, True])
def test_more_sequences_than_arrival_counters(hip, stream, drafted):
    rng = np.random.default_rng(11)
    n, vocab = 1500, 2500
    off = np.arange(n + 1, dtype=np.int32) * 2
    logits = (3 * rng.standard_normal((2 * n, vocab))).astype(np.float32)
    token = rng.integers(0, vocab, 2 * n)
    token[1::4] = logits[0::4].argmax(1)
    c = Case(logits, off, token, rng.random(2 * n).astype(np.float32), draft=softmax_rows(rng, 2 * n, vocab) if drafted else None,
             temperature=np.where(np.arange(n) % 5 == 0, 0.0, 0.8))
    assert c.check(c.run(hip, stream)) < n // 10


def test_temperatures_that_are_no_numbers(hip, stream):
    """Infinity has all tokens alike; what is below zero or no number counts as 0."""
    rng = np.random.default_rng(12)
    vocab, n = 1000, 8
    logits = rng.standard_normal((n, vocab)).astype(np.float32)
    logits[:, 500:] = -np.inf
    temperature = np.array([np.inf, np.inf, np.inf, -1.0, np.nan, -np.inf, 1e-45, 3e38], np.float32)
    u = np.array([0.0, 0.4991, 0.9999, 0.5, 0.5, 0.5, 0.5, 0.5011], np.float32)
    c = Case(logits, np.arange(n + 1, dtype=np.int32), np.zeros(n, int), u, temperature=temperature)
    n_path, _, tokens = c.run(hip, stream)
    assert (n_path == 1).all()
    best = logits.argmax(1)
    # (0.4991 x 500 = 249.55, 0.5011 x 500 = 250.55: no weight of 3e38 differs from 1 by 2^-100)
    assert tokens[:, 0].tolist() == [0, 249, 499, best[3], best[4], best[5], best[6], 250]


def test_verification_needs_parts(hip, stream):
    before = hip.alloc_stats().bytes_live
    ws = hip.workspace_create(2, 14, 64)
    whole = hip.alloc_stats().bytes_live - before
    hip.check(hip.mi_hip_workspace_destroy(ws))
    try:
        hip.check(hip.mi_hip_set_alloc_limit(before + whole - (1 << 20)))
        ws = hip.workspace_create(2, 14, 64)
    finally:
        hip.check(hip.mi_hip_set_alloc_limit(0))
    c = Case(np.zeros((2, 10), np.float32), np.array([0, 2], np.int32), np.zeros(2, int), np.zeros(2, np.float32))
    with pytest.raises(mh.MiHipError) as e:
        c.run(hip, stream, ws=ws)
    assert e.value.code == 5
    hip.check(hip.mi_hip_workspace_destroy(ws))


@pytest.mark.parametrize("in_place", [False, True])
def test_lengths_at_the_end_of_their_type(hip, stream, in_place):
    """Lengths whose sum passes 32 bits are refused, those around them are not."""
    from test_page_tables_gpu import Call, same, state
    rng = np.random.default_rng(13)
    big = 2 ** 31 - 1
    cached, new = np.array([5, big, 40, big - 14, 3]), np.array([3, 1, 1, 15, 7])
    s = state(rng, 5, 16, np.minimum(cached, 100), new, np.array([1, 2, 3, 0, 1]), 30)
    s["cached"] = cached
    c = Call(s, stream, in_place=in_place)
    hip.check(hip.mi_hip_page_tables(ctypes.byref(c.args)))
    same(c.got(), paged_ref.page_tables(**s))
