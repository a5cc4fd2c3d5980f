"""Attention over pages (mi_hip_attn_paged) against 64 bits; the tolerance is derived in
serve_ref.attention_tolerance. Rows of the pool that no query sees hold NaN and infinities."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref
from test_kv8_gpu import dev

pytestmark = pytest.mark.gpu

KINDS = {"f32": mh.MI_TYPE_F32, "f16": mh.MI_TYPE_F16, "q8": mh.MI_HIP_TYPE_Q8}


class Batch:
    """Sequences of (n_kv, new) over a pool whose pages are dealt in any order."""

    def __init__(self, hip, rng, cache, d, hkv, rep, page, seqs, lead=0, tail=0, scale=None, qmul=1.0, kmul=1.0, extra_pages=2):
        import torch
        self.hip, self.d, self.hkv, self.rep, self.page, self.seqs = hip, d, hkv, rep, page, seqs
        self.scale = float(np.float32(d ** -0.5 if scale is None else scale))
        pages = [-(-max(n, 0) // page) for n, _ in seqs]
        n_pages = sum(pages) + extra_pages
        ids = rng.permutation(n_pages)
        self.table = np.full((len(seqs), max(pages + [1]) + 1), -1, np.int32)
        at = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = ids[at:at + n]
            at += n
        rows = n_pages * page
        k, v = ((rng.standard_normal((rows, hkv, d)) * m).astype(np.float32) for m in (kmul, 1.0))
        live = np.zeros(rows, bool)
        for i, (n, _) in enumerate(seqs):
            live[self.rows_of(i)] = True
        k[~live], v[~live] = np.nan, np.inf
        if cache == "f16":
            k, v = k.astype(np.float16).astype(np.float32), v.astype(np.float16).astype(np.float32)
        self.kv = hip.kv_create_paged(2, n_pages, page, hkv, d, hkv * rep, KINDS[cache])
        for w, x in enumerate((k, v)):
            hip.kv_write(self.kv, 1, w, 0, dev(x), None)
        if cache == "q8":
            k, v = ref.q8(k, 0), ref.q8(v, 1)
        self.k, self.v = k, v
        new = [n for _, n in seqs]
        self.q_off = (lead + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
        self.t = int(self.q_off[-1]) + tail
        self.q = (rng.standard_normal((self.t, hkv * rep, d)) * qmul).astype(np.float32)
        self.dq, self.dtable, self.dq_off = dev(self.q), dev(self.table), dev(self.q_off)
        self.dn_kv = dev(np.array([n for n, _ in seqs], np.int32))
        self.out = torch.full(self.q.shape, 7.5, device="cuda")

    def rows_of(self, i):
        n = max(self.seqs[i][0], 0)
        t = np.arange(n)
        return self.table[i, t // self.page].astype(np.int64) * self.page + t % self.page

    def args(self, stream, **kw):
        return mh.paged_attn_args(self.kv, 1, self.dq, self.out, self.dq_off, self.dn_kv, self.dtable, self.scale, stream, **kw)

    def run(self, stream, **kw):
        import torch
        self.hip.check(self.hip.mi_hip_attn_paged(ctypes.byref(self.args(stream, **kw))))
        torch.cuda.synchronize()
        return self.out.cpu().numpy().astype(np.float64)

    def check(self, got, what="", skip=()):
        mine = np.zeros(self.t, bool)
        for i, (n, new) in enumerate(self.seqs):
            r0, r1 = self.q_off[i], self.q_off[i + 1]
            mine[r0:r1] = True
            if i in skip or new == 0:
                continue
            rows = self.rows_of(i)
            k, v = self.k[rows], self.v[rows]
            seen = np.arange(len(rows))[None, :] <= (n - new + np.arange(new))[:, None]
            want = ref.attention(self.q[r0:r1], k, v, seen, self.scale) if len(rows) else np.zeros((new,) + self.q.shape[1:])
            tol = ref.attention_tolerance(self.q[r0:r1], k, v, seen, self.scale) if len(rows) else 0.0
            assert np.isfinite(got[r0:r1]).all(), f"{what} sequence {i}: not finite"
            err = np.abs(got[r0:r1] - want).max()
            assert err <= tol, f"{what} sequence {i} ({n}, {new}): {err:.3e} > {tol:.3e}"
            assert (got[r0:r1][~seen.any(1)] == 0.0).all()
        assert (got[~mine] == 7.5).all(), f"{what}: rows of no sequence"

    def close(self):
        self.hip.check(self.hip.mi_hip_kv_destroy(self.kv))


BATCHES = [  # head_dim, kv heads, heads per kv head, page, sequences (n_kv, new)
    (64, 2, 7, 16, [(1, 1)]),
    (128, 4, 7, 16, [(500, 1)]),
    (64, 1, 1, 32, [(33, 1), (16, 1), (1, 1), (17, 1)]),
    (64, 2, 7, 16, [(0, 0), (40, 3), (0, 0), (31, 1)]),
    (128, 2, 4, 64, [(129, 6), (64, 8), (63, 5)]),
    (128, 1, 8, 16, [(70, 5), (3, 3), (300, 33)]),
    (64, 3, 5, 128, [(200, 200), (1, 1), (131, 64)]),
    (128, 4, 7, 16, [(1500, 25), (900, 1), (40, 1)]),
    (64, 2, 7, 256, [(3000, 1), (2047, 300), (5, 5), (257, 1)]),
    (64, 1, 16, 16, [(95, 2), (200, 40)]),
    (128, 1, 3, 32, [(700, 130), (2, 1), (33, 33), (32, 32), (31, 31)]),
    (64, 4, 2, 16, [(2, 5), (0, 3), (3, 100), (0, 40)]),  # more queries than positions: some see nothing
]


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("batch", BATCHES, ids=lambda b: "-".join(map(str, b[:4])) + f"-{len(b[4])}seq")
def test_against_64_bits(hip, stream, cache, batch):
    d, hkv, rep, page, seqs = batch
    b = Batch(hip, np.random.default_rng([d, hkv, rep, page, len(seqs)]), cache, d, hkv, rep, page, seqs, lead=2, tail=3)
    got = b.run(stream)
    b.check(got, str(batch))
    assert np.array_equal(got, b.run(stream))  # the same bits again
    b.check(b.run(stream, max_new=max(n for _, n in seqs)), "max_new")
    b.close()


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("d,hkv,rep", [(64, 2, 7), (128, 4, 7), (128, 1, 2)])
def test_many_ragged_sequences(hip, stream, cache, d, hkv, rep):
    rng = np.random.default_rng([d, rep])
    seqs = []
    for i in range(150):
        new = int(rng.choice([0, 1, 1, 1, 1, 3, 6, 20]))
        seqs.append((int(rng.choice([0, 5, 100, 333, 700])) + new, new))
    b = Batch(hip, rng, cache, d, hkv, rep, 16, seqs)
    b.check(b.run(stream))
    b.close()


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("n", [1, 7, 1100])
def test_more_sequences_than_a_wave(hip, stream, cache, n):
    rng = np.random.default_rng(n)
    seqs = [(int(rng.integers(1, 40)), 1) for _ in range(n)]
    b = Batch(hip, rng, cache, 64, 1, 4, 16, seqs)
    b.check(b.run(stream))
    b.check(b.run(stream, max_new=1))
    b.close()


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("seqs", [[(9000, 1)], [(5000, 1), (20000, 2)], [(6000, 40)], [(4200, 100), (15000, 1), (700, 700)]])
def test_long_sequences(hip, stream, cache, seqs):
    # (many workgroups share a sequence's keys and join their parts)
    b = Batch(hip, np.random.default_rng(len(seqs)), cache, 64, 2, 7, 64, seqs)
    got = b.run(stream)
    b.check(got)
    assert np.array_equal(got, b.run(stream))
    b.close()


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("qmul,kmul", [(40.0, 10.0), (1e-3, 1.0), (1e4, 1e-4)])
def test_scores_of_any_size(hip, stream, cache, qmul, kmul):
    b = Batch(hip, np.random.default_rng(3), cache, 128, 2, 4, 32, [(300, 1), (170, 20)], qmul=qmul, kmul=kmul)
    b.check(b.run(stream))
    b.close()


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("new", [1, 40])
def test_values_that_are_not_finite(hip, stream, cache, new):
    """NaN in a value row: the queries before it do not show it, those that see it do."""
    import torch
    n = 150
    b = Batch(hip, np.random.default_rng(5), cache, 64, 1, 4, 16, [(n, new), (90, 3)])
    want = b.run(stream)
    b.check(want)
    row = b.rows_of(0)[n - 1 - new // 2]
    x = torch.full((1, 1, 64), float("nan"), device="cuda")
    hip.kv_write(b.kv, 1, 1, int(row), x, None)
    got = b.run(stream)
    first = new - 1 - new // 2  # the first query that sees it
    assert np.array_equal(got[:first], want[:first]) and np.isnan(got[first:new]).all()
    assert np.array_equal(got[new:], want[new:])
    b.close()


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("page_id", [-1, 2 ** 31 - 1, None])
def test_tables_that_name_no_page(hip, stream, cache, new, page_id):
    # positions 32.. of sequence 0: those that see them get NaN, nobody else notices
    b = Batch(hip, np.random.default_rng(6), cache, 128, 2, 2, 16, [(60, new), (90, 3), (100, 50)])
    want = b.run(stream)
    b.dtable[0, 2] = len(b.k) // 16 if page_id is None else page_id
    got = b.run(stream)
    sees = 60 - new + np.arange(new) >= 32
    assert np.isnan(got[:new][sees]).all() and np.array_equal(got[:new][~sees], want[:new][~sees])
    assert np.array_equal(got[new:], want[new:])
    b.close()


def test_lengths_out_of_range(hip, stream):
    # offsets and lengths that no batch has: clamped, nothing outside is touched
    import torch
    b = Batch(hip, np.random.default_rng(7), "f16", 64, 2, 3, 16, [(100, 4), (50, 2), (70, 60)], tail=5)
    want = b.run(stream)
    b.dn_kv[1] = 2 ** 31 - 1  # as many as the table's row has; its entries behind are -1
    got = b.run(stream)
    assert np.isnan(got[4:6]).all() and np.array_equal(np.delete(got, [4, 5], 0), np.delete(want, [4, 5], 0))
    b.dn_kv[1] = -3
    assert (b.run(stream)[4:6] == 0).all()
    b.dn_kv[1] = 50
    b.dq_off.copy_(dev(np.array([-5, 4, 6, 2 ** 31 - 1], np.int32)))
    b.run(stream)  # (rows 0 .. 3 and 6 .. end)
    b.dq_off.copy_(dev(np.array([9, 4, 60, 3], np.int32)))
    b.run(stream)
    b.dq_off.copy_(dev(b.q_off))
    b.out.fill_(7.5)
    assert np.array_equal(b.run(stream), want)
    # queries beyond max_new are left as they were
    b.out.fill_(7.5)
    got = b.run(stream, max_new=3)
    keep = np.array([0, 1, 2, 4, 5, 6, 7, 8])
    assert (np.delete(got, keep, 0) == 7.5).all()
    b.check(np.where(np.isin(np.arange(b.t), keep)[:, None, None], got, want))
    torch.cuda.synchronize()
    b.close()


def test_strides(hip, stream):
    import torch
    b = Batch(hip, np.random.default_rng(8), "f16", 64, 2, 3, 16, [(100, 4), (300, 50), (7, 1)])
    want = b.run(stream)
    wide_q = torch.full((b.t, 9, 68), float("nan"), device="cuda")
    wide_q[:, 2:8, :64] = b.dq
    wide_o = torch.full((b.t, 8, 72), 7.5, device="cuda")
    table = torch.full((3, b.dtable.shape[1] + 6), -9, dtype=torch.int32, device="cuda")
    table[:, :b.dtable.shape[1]] = b.dtable
    a = mh.paged_attn_args(b.kv, 1, wide_q[:, 2:8, :64], wide_o[:, 1:7, 4:68], b.dq_off, b.dn_kv, table[:, :b.dtable.shape[1]],
                           b.scale, stream)
    hip.check(hip.mi_hip_attn_paged(ctypes.byref(a)))
    torch.cuda.synchronize()
    got = wide_o.cpu().numpy()
    assert np.array_equal(got[:, 1:7, 4:68].astype(np.float64), want)
    got[:, 1:7, 4:68] = 7.5
    assert (got == 7.5).all()
    b.close()


def test_two_streams_with_workspaces_of_their_own(hip, stream):
    import torch
    ws = [hip.workspace_create(2, 14, 64) for _ in range(2)]
    b = Batch(hip, np.random.default_rng(9), "f16", 64, 2, 7, 16, [(5000, 1), (3000, 40)])
    b.check(b.run(stream))
    want = b.run(stream, ws=ws[0])  # (another workspace may cut the keys otherwise)
    b.check(want)
    outs, streams = [torch.full_like(b.out, 7.5) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for o, s, w in zip(outs, streams, ws):
            a = mh.paged_attn_args(b.kv, 1, b.dq, o, b.dq_off, b.dn_kv, b.dtable, b.scale, s.cuda_stream, ws=w)
            hip.check(hip.mi_hip_attn_paged(ctypes.byref(a)))
    torch.cuda.synchronize()
    for o in outs:
        assert np.array_equal(o.cpu().numpy().astype(np.float64), want)
    for w in ws:
        hip.check(hip.mi_hip_workspace_destroy(w))
    b.close()


def test_graph_replays_read_the_lengths(hip, stream):
    """Two captured steps that share the cache's workspace, replayed on changing lengths and tables."""
    import torch
    rng = np.random.default_rng(10)
    b = Batch(hip, rng, "q8", 64, 2, 7, 16, [(3000, 2), (500, 2), (200, 100), (4, 2)])
    b.run(stream)
    side, outs = torch.cuda.Stream(), [torch.full_like(b.out, 7.5) for _ in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a = mh.paged_attn_args(b.kv, 1, b.dq, o, b.dq_off, b.dn_kv, b.dtable, b.scale, side.cuda_stream)
            hip.check(hip.mi_hip_attn_paged(ctypes.byref(a)))
        graphs.append(g)
    for step in range(4):
        n = np.array([int(rng.integers(1, 3001)), int(rng.integers(2, 501)), int(rng.integers(100, 201)), 4])
        b.seqs = [(int(x), new) for x, (_, new) in zip(n, b.seqs)]
        b.dn_kv.copy_(dev(n.astype(np.int32)))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        eager = b.run(stream)
        b.check(eager)
        for o in outs:
            assert np.array_equal(o.cpu().numpy().astype(np.float64), eager)
    b.close()


def test_refusals(hip, stream):
    import torch
    b = Batch(hip, np.random.default_rng(11), "f16", 64, 2, 3, 16, [(100, 4)])
    plain = hip.kv_create(2, 48, 2, 64, 6, mh.MI_TYPE_F16)

    def rc(**kw):
        a = b.args(stream)
        for n, v in kw.items():
            if n in ("q_nb", "out_nb"):
                getattr(a, n)[:] = v
            else:
                setattr(a, n, v)
        return hip.mi_hip_attn_paged(ctypes.byref(a))
    nb = mh.nb3_of(b.dq)
    for kw, code in ((dict(kv=plain), 5), (dict(layer=2), 1), (dict(n_seq=-1), 1), (dict(n_tokens=-1), 1), (dict(max_new=-1), 1),
                     (dict(max_pages=0), 1), (dict(n_head=5), 1), (dict(n_head=0), 1), (dict(n_tokens=1 << 25), 5),
                     (dict(max_pages=1 << 27, table_nb=1 << 29), 5), (dict(n_seq=(1 << 20) + 1), 5), (dict(scale=float("nan")), 1),
                     (dict(q_off=None), 1), (dict(n_kv=None), 1), (dict(table=None), 1), (dict(q=None), 1), (dict(out=None), 1),
                     (dict(table=b.dtable.data_ptr() + 2), 1), (dict(n_seq=2, table_nb=4), 1), (dict(table_nb=6), 1),
                     (dict(q_nb=(8, nb[1], nb[2])), 5), (dict(out_nb=(4, nb[1] + 4, nb[2])), 5), (dict(q=b.dq.data_ptr() + 4), 5)):
        assert rc(**kw) == code, (kw, hip.last_error())
    assert rc(n_seq=0) == 0 and rc(n_tokens=0) == 0
    torch.cuda.synchronize()
    assert (b.out == 7.5).all()
    hip.check(hip.mi_hip_kv_destroy(plain))
    b.close()


@pytest.mark.parametrize("new", [1, 60])
def test_offsets_at_the_end_of_their_type(hip, stream, new):
    """An offset of -2^31 counts as 0: the sequence that ends there has no queries, the next one begins at row 0.
    max_new reaches beyond the rows that there are, which guards hold."""
    import torch
    b = Batch(hip, np.random.default_rng(14), "f16", 64, 2, 3, 16, [(100, 4), (50, 2), (90, new)])
    rows = b.t - 2
    guarded = torch.full((rows + 80,) + tuple(b.out.shape[1:]), 7.5, device="cuda")
    q = torch.zeros_like(guarded)
    q[:rows] = b.dq[:rows]
    outs = []
    for low in (0, -1, -2 ** 31, -2 ** 31 + 3):
        b.dq_off.copy_(dev(np.array([6, low, 4, rows], np.int32)))
        guarded.fill_(7.5)
        a = mh.paged_attn_args(b.kv, 1, q[:rows], guarded[:rows], b.dq_off, b.dn_kv, b.dtable, b.scale, stream,
                               max_new=0 if new == 1 else 64)
        hip.check(hip.mi_hip_attn_paged(ctypes.byref(a)))
        torch.cuda.synchronize()
        outs.append(guarded.cpu().numpy())
        assert (outs[-1][rows:] == 7.5).all()
        assert all(np.array_equal(x, outs[0]) for x in outs)
    b.close()


@pytest.mark.parametrize("n_kv,new", [(16, 9000000), (40, 5000), (300, 2000)])
def test_far_more_queries_than_positions(hip, stream, n_kv, new):
    """The queries that see no position give zeros, however many they are; the last ones see theirs."""
    import torch
    b = Batch(hip, np.random.default_rng(15), "f16", 64, 1, 1, 16, [(n_kv, n_kv)])
    last = dev(b.q)
    q = last[-1:].expand(new, 1, 64)  # (every query the same row, which takes no memory)
    out = torch.full((new, 1, 64), 7.5, device="cuda")
    a = mh.paged_attn_args(b.kv, 1, q, out, dev(np.array([0, new], np.int32)), b.dn_kv, b.dtable[:, :-(-n_kv // 16)], b.scale, stream)
    hip.check(hip.mi_hip_attn_paged(ctypes.byref(a)))
    torch.cuda.synchronize()
    assert bool((out[:new - n_kv] == 0).all())
    b.q = np.repeat(b.q[-1:], n_kv, 0)
    b.check(out[new - n_kv:].cpu().numpy().astype(np.float64))
    b.close()
