"""Steps of a server over a paged cache as the integration guide describes them: sequences that are refused
for want of pages, prompts among chains of drafted tokens, and pages that sequences share."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import paged_ref
import serve_ref as ref
from test_kv8_gpu import dev
from test_paged_step_gpu import KINDS, PAGE, Server

pytestmark = pytest.mark.gpu


def check_attention(s, layer, i, n_kv, rows, stream, what):
    """Sequence i's outputs against 64 bits over its rows of the pool."""
    new = rows.stop - rows.start
    k, v = (s.rows(layer, w, i, n_kv, stream) for w in (0, 1))
    seen = np.arange(n_kv)[None, :] <= (n_kv - new + np.arange(new))[:, None]
    q = s.qr[layer, rows].cpu().numpy()
    err = np.abs(s.out[layer, rows].cpu().numpy() - ref.attention(q, k, v, seen, s.scale)).max()
    assert err <= ref.attention_tolerance(q, k, v, seen, s.scale), what


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("n_pages", [22, 30])
def test_refused_sequences_and_prompts_among_chains(hip, stream, kind, captured, n_pages):
    """A pool too small for all: a refused sequence stays where it is until it is granted, a prompt's chunk
    moves on by its length, a chain by what was accepted. Every step reads, in the rows before its own,
    what the steps before it have stored."""
    import torch
    n, most, chunk, d, hkv, rep, vocab = 8, 6, 50, 64, 2, 7, 700
    s = Server(hip, kind, n, n_pages, n * chunk, 12, d, hkv, rep, 1, most, vocab, 9)
    i32 = lambda *x: torch.zeros(x, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    # the nodes to verify: all rows of a chain, the last one of a prompt's chunk
    nodes, off, node_token, prompt = n * most, i32(n + 1), i32(n * most), i32(n)
    row = torch.zeros(nodes, dtype=torch.int64, device="cuda")
    logits, u = torch.zeros(nodes, vocab, device="cuda"), torch.zeros(nodes, device="cuda")

    def step(st):
        s.place(st)
        s.attend(st, max_new=chunk)
        torch.index_select(s.logits, 0, row, out=logits)
        a = mh.verify_args(logits, off, node_token, u, s.n_path, s.path, s.tokens, st, temperature=s.temperature, ws=s.ws)
        hip.check(hip.mi_hip_verify_draft(ctypes.byref(a)))
        moved = torch.where(prompt > 0, s.new, s.n_path)
        s.cached.add_(torch.where(s.n_kv > 0, moved, torch.zeros_like(moved)))

    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(side.cuda_stream)
    rng = np.random.default_rng([3, 1])
    s.temperature.fill_(1.0)
    stored = [None] * n  # K and V rows of each sequence's certain tokens
    cached, waits = np.zeros(n, int), np.zeros(n, bool)
    waited = 0
    for turn in range(24):
        begins = cached == 0
        ends = (cached > 70) & ~waits & (rng.random(n) < 0.6)
        new = np.where(begins, rng.integers(20, chunk + 1, n), rng.integers(1, most + 1, n))
        cached[ends], new[ends], begins[ends] = 0, 0, False
        q_off = np.concatenate([[0], np.cumsum(new)])
        take = np.where(begins, np.minimum(new, 1), new)
        node_off = np.concatenate([[0], np.cumsum(take)])
        src = np.concatenate([np.arange(q_off[i + 1] - take[i], q_off[i + 1]) for i in range(n)])
        gen = torch.Generator(device="cuda").manual_seed(turn)
        for x in (s.q, s.k, s.v, s.logits):
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
        token = rng.integers(0, vocab, nodes)
        likely = rng.random(nodes) < 0.8  # drafts that are likely to be accepted
        for r in range(1, len(src)):
            if likely[r]:
                s.logits[int(src[r - 1]), int(token[r])] = 12.0
        fill = lambda t, x: t.copy_(dev(np.resize(x, t.shape).astype({torch.int64: np.int64, torch.int32: np.int32}[t.dtype])))
        fill(s.cached, cached), fill(s.new, new), fill(off, node_off), fill(prompt, begins), fill(node_token, token)
        fill(row, np.concatenate([src, np.zeros(nodes - len(src), int)]))
        u.copy_(torch.rand(nodes, device="cuda", generator=gen))
        torch.cuda.synchronize()
        if captured:
            graph.replay()
        else:
            step(stream)
        torch.cuda.synchronize()
        n_kv, n_path, after = (x.cpu().numpy() for x in (s.n_kv, s.n_path, s.cached))
        assert np.array_equal(s.q_off.cpu().numpy(), q_off)
        refused = (n_kv == 0) & (new > 0)
        assert s.refused.item() == refused.sum()
        for i in range(n):
            rows = slice(int(q_off[i]), int(q_off[i + 1]))
            if refused[i]:
                assert after[i] == cached[i]
                assert bool((s.out[0, rows] == 0).all()) and bool((s.slots[rows] == -1).all())
            elif new[i]:
                assert n_kv[i] == cached[i] + new[i]
                assert after[i] == cached[i] + (new[i] if begins[i] else n_path[i])
                k, v = (s.rows(0, w, i, int(n_kv[i]), stream) for w in (0, 1))
                if cached[i]:
                    assert all(np.array_equal(x[:cached[i]], y) for x, y in zip((k, v), stored[i])), (turn, i)
                check_attention(s, 0, i, int(n_kv[i]), rows, stream, (turn, i))
                path, _, margin = paged_ref.verify(*(x[node_off[i]:node_off[i + 1]] for x in (logits.cpu().numpy(), token)), None,
                                                   None, 1.0, u.cpu().numpy()[node_off[i]:node_off[i + 1]], most)
                assert margin < vocab * 2.0 ** -53 or n_path[i] == len(path)
                stored[i] = (k[:after[i]], v[:after[i]])
                waited += waits[i]
        waits = refused
        cached = after.astype(int)
        held, table, at = s.held.cpu().numpy(), s.table.cpu().numpy(), s.ring_at.cpu().numpy()
        free = s.ring.cpu().numpy()[np.arange(*at) % n_pages]
        assert np.array_equal(np.sort(np.concatenate([table[i, :held[i]] for i in range(n)] + [free])), np.arange(n_pages))
    assert waited > 0  # some were refused, and granted later
    s.close()


@pytest.mark.parametrize("kind", list(KINDS))
def test_pages_of_a_common_prompt(hip, stream, kind):
    """Two pages of a prompt stand in front of every table row and outside of what the tables' call manages: its
    rows begin behind them, and positions and lengths get theirs added. They are never given back or dealt."""
    import torch
    n, n_pages, lead, d, hkv, rep = 4, 30, 2, 64, 2, 7
    s = Server(hip, kind, n, n_pages, 60, 10, d, hkv, rep, 1, 6, 100, 4)
    ring = s.ring.cpu().numpy()
    shared, front = ring[:lead].copy(), lead * PAGE
    s.ring_at.copy_(dev(np.array([lead, n_pages], np.int32)))  # two pages are with the prompt
    s.table[:, :lead] = dev(shared)
    rng = np.random.default_rng(8)
    pk, pv = (rng.standard_normal((front, hkv, d)).astype(np.float32) for _ in range(2))
    slots = (shared[np.arange(front) // PAGE] * PAGE + np.arange(front) % PAGE).astype(np.int32)
    a = mh.paged_append_args(s.kv, 0, d, 1e6, stream, dev(pk), dev(pv), dev(slots), dev(np.arange(front, dtype=np.int32)), freq=s.freq,
                             k_norm=s.wk, eps=1e-6)
    hip.check(hip.mi_hip_paged_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    prompt = [s.rows(0, w, 0, front, stream) for w in (0, 1)]
    cached = np.zeros(n, int)  # without the prompt
    for turn in range(8):
        new = rng.integers(1, 16, n)
        if turn in (3, 5):  # requests end
            cached[turn % n], new[turn % n] = 0, 0
        s.cached.copy_(dev(cached.astype(np.int32)))
        s.new.copy_(dev(new.astype(np.int32)))
        gen = torch.Generator(device="cuda").manual_seed(turn)
        for x in (s.q, s.k, s.v):
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
        a = mh.page_tables_args(PAGE, s.cached, s.new, s.held, s.held, s.table[:, lead:], s.ring, s.ring_at, s.ring_at, s.n_kv,
                                s.q_off, s.slots, stream, pos=s.pos, n_refused=s.refused)
        hip.check(hip.mi_hip_page_tables(ctypes.byref(a)))
        s.pos.add_(front)
        s.n_kv.copy_(torch.where(s.n_kv > 0, s.n_kv + front, torch.zeros_like(s.n_kv)))
        s.attend(stream, max_new=15)
        torch.cuda.synchronize()
        assert s.refused.item() == 0
        off, n_kv = s.q_off.cpu().numpy(), s.n_kv.cpu().numpy()
        assert np.array_equal(n_kv, np.where(new > 0, front + cached + new, 0))
        for i in np.nonzero(new)[0]:
            rows = slice(int(off[i]), int(off[i + 1]))
            assert np.array_equal(s.pos.cpu().numpy()[rows], front + cached[i] + np.arange(new[i]))
            check_attention(s, 0, i, int(n_kv[i]), rows, stream, (turn, i))
            assert all(np.array_equal(s.rows(0, w, i, front, stream), prompt[w]) for w in (0, 1))
        cached += new
        held, table, at = s.held.cpu().numpy(), s.table.cpu().numpy(), s.ring_at.cpu().numpy()
        free = s.ring.cpu().numpy()[np.arange(*at) % n_pages]
        owned = np.concatenate([table[i, lead:lead + held[i]] for i in range(n)] + [free, shared])
        assert np.array_equal(np.sort(owned), np.arange(n_pages)) and (table[:, :lead] == shared).all()
    s.close()
