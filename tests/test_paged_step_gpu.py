"""The operators over a paged cache together, as a server with drafted tokens calls them: block tables,
append, attention, verification, and the next step from what was accepted. Checked against the same
tokens fed to a cache of each sequence's own (cache rows: bit for bit; attention: the rounding of sums,
serve_ref.attention_tolerance), and captured against eager (bit for bit)."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import paged_ref
import serve_ref as ref
from test_kv8_gpu import dev, read

pytestmark = pytest.mark.gpu

EPS, PAGE = 1e-6, 16
KINDS = {"f32": mh.MI_TYPE_F32, "f16": mh.MI_TYPE_F16, "q8": mh.MI_HIP_TYPE_Q8}


class Server:
    """A pool, the lists of the sequences that share it, and the framework's calls of one step."""

    def __init__(self, hip, kind, n, n_pages, max_tokens, max_pages, d, hkv, rep, layers, max_path, vocab, seed):
        import torch
        rng = np.random.default_rng(seed)
        self.hip, self.d, self.hkv, self.h, self.layers, self.n = hip, d, hkv, hkv * rep, layers, n
        self.n_pages, self.max_tokens = n_pages, max_tokens
        self.scale = float(np.float32(d ** -0.5))
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.kv = hip.kv_create_paged(layers, n_pages, PAGE, hkv, d, self.h, KINDS[kind])
        self.ws = hip.workspace_create(hkv, hkv * rep, d)
        self.ring, self.ring_at = dev(rng.permutation(n_pages).astype(np.int32)), dev(np.array([0, n_pages], np.int32))
        self.cached, self.new, self.held, self.n_kv, self.n_path = (i32(n) for _ in range(5))
        self.table, self.q_off = i32(n, max_pages), i32(n + 1)
        self.slots, self.pos, self.token, self.refused = i32(max_tokens), i32(max_tokens), i32(max_tokens), i32(1)
        self.path, self.tokens = i32(n, max_path), i32(n, max_path)
        f32 = lambda *s: torch.zeros(s, device="cuda")
        self.q, self.qr, self.out = (f32(layers, max_tokens, self.h, d) for _ in range(3))
        self.k, self.v = (f32(layers, max_tokens, hkv, d) for _ in range(2))
        self.logits, self.u, self.temperature = f32(max_tokens, vocab), f32(max_tokens), f32(n)
        self.freq = (1e6 ** (-np.arange(0, d, 2, dtype=np.float64) / d)).astype(np.float32)
        self.wq, self.wk = (dev((1 + 0.2 * rng.standard_normal(d)).astype(np.float32)) for _ in range(2))

    def place(self, stream):
        a = mh.page_tables_args(PAGE, self.cached, self.new, self.held, self.held, self.table, self.ring, self.ring_at,
                                self.ring_at, self.n_kv, self.q_off, self.slots, stream, pos=self.pos, n_refused=self.refused)
        self.hip.check(self.hip.mi_hip_page_tables(ctypes.byref(a)))

    def attend(self, stream, max_new=0):
        for layer in range(self.layers):
            a = mh.paged_append_args(self.kv, layer, self.d, 1e6, stream, self.k[layer], self.v[layer], self.slots, self.pos,
                                     q=self.q[layer], q_out=self.qr[layer], freq=self.freq, q_norm=self.wq, k_norm=self.wk,
                                     eps=EPS)
            self.hip.check(self.hip.mi_hip_paged_append(ctypes.byref(a)))
            a = mh.paged_attn_args(self.kv, layer, self.qr[layer], self.out[layer], self.q_off, self.n_kv, self.table, self.scale,
                                   stream, max_new=max_new)
            self.hip.check(self.hip.mi_hip_attn_paged(ctypes.byref(a)))

    def verify(self, stream):
        a = mh.verify_args(self.logits, self.q_off, self.token, self.u, self.n_path, self.path, self.tokens, stream,
                           temperature=self.temperature, ws=self.ws)
        self.hip.check(self.hip.mi_hip_verify_draft(ctypes.byref(a)))

    def rows(self, layer, which, i, n, stream):
        """Sequence i's first n rows of the pool."""
        pool = read(self.hip, self.kv, layer, which, 0, self.n_pages * PAGE, self.hkv, self.d, stream)
        t, table = np.arange(n), self.table[i].cpu().numpy()
        return pool[table[t // PAGE].astype(np.int64) * PAGE + t % PAGE]

    def close(self):
        self.hip.check(self.hip.mi_hip_workspace_destroy(self.ws))
        self.hip.check(self.hip.mi_hip_kv_destroy(self.kv))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d,hkv,rep", [(64, 2, 7), (128, 2, 4)])
def test_steps_against_sequences_of_their_own(hip, stream, kind, d, hkv, rep):
    import torch
    rng = np.random.default_rng([d, list(KINDS).index(kind)])
    prompts, layers, vocab, drafted = [70, 1, 33, 17, 150], 2, 500, 3
    n = len(prompts)
    s = Server(hip, kind, n, 64, sum(prompts), 20, d, hkv, rep, layers, 1 + drafted, vocab, [d, 3])
    s.temperature.copy_(dev(np.array([0.0, 1.0, 0.3, 0.7, 2.0], np.float32)))
    emb = [[dev(rng.standard_normal((vocab, heads, d)).astype(np.float32)) for heads in (s.h, hkv, hkv)] for _ in range(layers)]
    head = dev((rng.standard_normal((vocab, s.h * d)) * 0.3).astype(np.float32))
    said = [list(rng.integers(0, vocab, p)) for p in prompts]  # all certain tokens
    cached, accepted = np.zeros(n, int), 0
    for step in range(6):
        feed = [x[cached[i]:] for i, x in enumerate(said)]
        if step:  # drafts: the likely successors of the last certain token
            for f in feed:
                for _ in range(drafted):
                    f.append((7 * f[-1] + 1) % vocab)
        new = np.array([len(f) for f in feed])
        flat = np.concatenate(feed)
        t = len(flat)
        s.new.copy_(dev(new.astype(np.int32)))
        s.token.zero_()
        s.token[:t] = dev(flat.astype(np.int32))
        for layer in range(layers):
            for x, e in zip((s.q, s.k, s.v), emb[layer]):
                x[layer] = e[s.token.long()]
        s.u.copy_(torch.from_numpy(rng.random(s.max_tokens).astype(np.float32)))
        s.place(stream)
        s.attend(stream, max_new=int(new.max()))
        torch.mm(s.out[-1].view(s.max_tokens, -1), head.t(), out=s.logits)
        likely = (7 * s.token.long() + 1) % vocab
        s.logits[torch.arange(s.max_tokens, device="cuda"), likely] = s.logits.max(1).values + 1.0
        torch.cuda.synchronize()
        assert s.refused.item() == 0
        off, n_kv = s.q_off.cpu().numpy(), s.n_kv.cpu().numpy()
        assert np.array_equal(off, np.concatenate([[0], np.cumsum(new)])) and np.array_equal(n_kv, cached + new)
        # the attention, from the rows in the cache
        for layer in range(layers):
            for i in range(n):
                k, v = (s.rows(layer, w, i, n_kv[i], stream) for w in (0, 1))
                seen = np.arange(n_kv[i])[None, :] <= (cached[i] + np.arange(new[i]))[:, None]
                q = s.qr[layer, off[i]:off[i + 1]].cpu().numpy()
                err = np.abs(s.out[layer, off[i]:off[i + 1]].cpu().numpy() - ref.attention(q, k, v, seen, s.scale)).max()
                assert err <= ref.attention_tolerance(q, k, v, seen, s.scale), (step, layer, i)
        if step == 0:  # a prompt: its last row alone is drawn from
            s.q_off.copy_(dev(np.arange(n + 1).astype(np.int32)))
            last = torch.from_numpy(off[1:] - 1).cuda().long()
            s.logits[:n] = s.logits[last]
            off = np.arange(n + 1)
        s.verify(stream)
        torch.cuda.synchronize()
        logits, u, n_path = s.logits.cpu().numpy(), s.u.cpu().numpy(), s.n_path.cpu().numpy()
        token, temperature = s.token.cpu().numpy(), s.temperature.cpu().numpy()
        for i in range(n):
            r = slice(off[i], off[i + 1])
            path, tokens, margin = paged_ref.verify(logits[r], token[r], None, None, temperature[i], u[r], 1 + drafted)
            got = s.tokens[i].cpu().numpy()[:n_path[i]].tolist()
            if margin >= vocab * 2.0 ** -53:
                assert got == tokens and s.path[i].cpu().numpy()[:n_path[i]].tolist() == path
            said[i] += got
            accepted += n_path[i] - 1
            cached[i] += n_path[i] if step else prompts[i]
        s.cached.copy_(dev(cached.astype(np.int32)))
        assert [len(x) for x in said] == (cached + 1).tolist()
    assert accepted >= 5 * drafted  # the greedy sequence accepts all of its drafts
    # the same tokens, a cache for each sequence
    for i in range(n):
        one = hip.kv_create(layers, cached[i], hkv, d, s.h, KINDS[kind])
        toks = torch.tensor(said[i][:cached[i]], device="cuda")
        for layer in range(layers):
            a = mh.norm_rope_args(one, layer, 0, d, 1e6, stream, emb[layer][1][toks], emb[layer][2][toks], freq=s.freq, k_norm=s.wk,
                                  eps=EPS)
            hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
            torch.cuda.synchronize()
            for w in (0, 1):
                assert np.array_equal(read(hip, one, layer, w, 0, int(cached[i]), hkv, d, stream),
                                      s.rows(layer, w, i, int(cached[i]), stream)), (i, layer, w)
        hip.check(hip.mi_hip_kv_destroy(one))
    s.close()


@pytest.mark.parametrize("kind", list(KINDS))
def test_captured_step(hip, stream, kind):
    """A whole step as a graph, replayed on lengths that its own outputs set; an eager twin, between the
    replays, gives the same bits. Nothing allocates."""
    import torch
    n, d, hkv, rep, layers, vocab, most = 9, 64, 2, 7, 2, 3001, 6
    shape = (n, 120, n * most, 16, d, hkv, rep, layers, most, vocab)
    twins = [Server(hip, kind, *shape, 7) for _ in range(2)]

    def step(s, st):
        s.place(st)
        s.attend(st, max_new=most)
        s.verify(st)
        s.cached.add_(s.n_path)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(twins[0], side.cuda_stream)
    before = hip.alloc_stats()
    rng = np.random.default_rng(5)
    names = ("cached", "held", "table", "ring", "ring_at", "n_kv", "q_off", "slots", "pos", "refused", "n_path", "path", "tokens",
             "qr", "out")
    for turn in range(12):
        new = rng.integers(0 if turn else 1, most + 1, n).astype(np.int32)
        ended = rng.random(n) < (0.1 if turn else 0.0)
        gen = torch.Generator(device="cuda").manual_seed(turn)
        fresh = {x: torch.randn(getattr(twins[0], x).shape, device="cuda", generator=gen) for x in ("q", "k", "v", "logits")}
        # a likely token in most places, so that drafts are accepted
        token = torch.randint(vocab, (n * most,), device="cuda", generator=gen).int()
        fresh["logits"][torch.arange(n * most - 1, device="cuda"), token[1:].long()] = 9.0
        u = torch.rand(n * most, device="cuda", generator=gen)
        for s in twins:
            for x, value in fresh.items():
                getattr(s, x).copy_(value)
            s.token.copy_(token)
            s.u.copy_(u)
            s.new.copy_(dev(np.where(ended, 0, new).astype(np.int32)))
            s.cached[torch.from_numpy(ended).cuda()] = 0
            s.temperature.fill_(1.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(twins[1], stream)
        torch.cuda.synchronize()
        for x in names:
            assert torch.equal(getattr(twins[0], x), getattr(twins[1], x)), (turn, x)
        held, table = twins[1].held.cpu().numpy(), twins[1].table.cpu().numpy()
        at = twins[1].ring_at.cpu().numpy()
        free = twins[1].ring.cpu().numpy()[np.arange(*at) % 120]
        assert np.array_equal(np.sort(np.concatenate([table[i, :held[i]] for i in range(n)] + [free])), np.arange(120))
    assert int(twins[0].cached.max()) > PAGE  # a second page was taken
    for layer in range(layers):
        for w in (0, 1):
            a, b = (read(hip, s.kv, layer, w, 0, 120 * PAGE, hkv, d, stream, half=True) for s in twins)
            assert np.array_equal(a, b, equal_nan=True)
    after = hip.alloc_stats()
    assert (after.n_malloc, after.n_free) == (before.n_malloc, before.n_free)
    for s in twins:
        s.close()
