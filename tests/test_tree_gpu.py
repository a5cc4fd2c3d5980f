"""Attention of drafted tokens (mi_hip_attn_tree) against 64 bits.

The cache is read back (or known) exactly, so the reference takes the same
values; the tolerance is derived in serve_ref.attention_tolerance.
"""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref

pytestmark = pytest.mark.gpu

CACHES = ["f32", "f16", "q8"]


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def dev_bits(bits):
    return None if bits is None else dev(bits.view(np.int64))


class Seq:
    """One sequence: its cache (a handle for q8, tensors otherwise), queries, mask and reference."""

    def __init__(self, hip, rng, cache, d, hkv, rep, n_past, t, bits, spare=3, scale=None, qmul=1.0, k=None, v=None):
        import torch
        self.hip, self.n_past, self.t, self.rep, self.bits = hip, n_past, t, rep, bits
        n = n_past + t
        self.scale = float(np.float32(d ** -0.5 if scale is None else scale))
        self.q = (rng.standard_normal((t, hkv * rep, d)) * qmul).astype(np.float32)
        k = rng.standard_normal((n + spare, hkv, d)).astype(np.float32) if k is None else k
        v = rng.standard_normal((n + spare, hkv, d)).astype(np.float32) if v is None else v
        k[n:], v[n:] = np.nan, np.inf  # rows behind the last are stale: never seen
        self.kv = None
        if cache == "q8":
            self.kv = hip.kv_create(1, n + spare, hkv, d, hkv * rep, mh.MI_HIP_TYPE_Q8)
            for w, x in enumerate((k, v)):
                hip.kv_write(self.kv, 0, w, 0, dev(x), None)
            self.src = dict(kv=self.kv, layer=0)
            k, v = ref.q8(k, 0), ref.q8(v, 1)
        else:
            dt = np.float16 if cache == "f16" else np.float32
            k, v = k.astype(dt), v.astype(dt)
            self.dk, self.dv = dev(k), dev(v)
            self.src = dict(k=self.dk, v=self.dv)
        self.k, self.v = k[:n], v[:n]
        self.dq, self.dbits = dev(self.q), dev_bits(bits)
        self.out = torch.full(self.dq.shape, float("nan"), device="cuda")

    def args(self, stream, ws=None):
        return mh.attn_args(self.dq, self.out, self.rep, self.n_past, self.scale, stream, ws=ws, **self.src)

    def check(self, what):
        got = self.out.cpu().numpy().astype(np.float64)
        seen = ref.visible(self.n_past, self.t, self.bits)
        k, v = self.k.astype(np.float64), self.v.astype(np.float64)
        want = ref.attention(self.q, np.where(np.isfinite(k), k, 0), np.where(np.isfinite(v), v, 0), seen, self.scale)
        tol = ref.attention_tolerance(self.q, np.where(np.isfinite(k), k, 0), np.where(np.isfinite(v), v, 0), seen,
                                      self.scale)
        assert np.all(np.isfinite(got)), f"{what}: not finite"
        err = np.abs(got - want).max(initial=0.0)
        assert err <= tol, f"{what}: {err:.3e} > {tol:.3e}"
        empty = ~seen.any(1)
        assert np.all(got[empty] == 0.0), f"{what}: rows that see nothing"

    def close(self):
        if self.kv:
            import torch
            torch.cuda.synchronize()
            self.hip.check(self.hip.mi_hip_kv_destroy(self.kv))


def run(hip, seqs, stream, ws=None):
    import torch
    items = (mh.AttnArgs * len(seqs))(*[s.args(stream, ws) for s in seqs])
    masks = mh.tree_masks([s.dbits for s in seqs])
    hip.check(hip.mi_hip_attn_tree(items, masks, len(seqs), stream))
    torch.cuda.synchronize()


def make_bits(rng, kind, t):
    words = (t + 63) // 64
    if kind == "chain":
        return None
    if kind == "tree":
        return ref.random_tree(rng, t)[0]
    if kind == "none":  # every row empty of drafted keys
        return np.zeros((t, words), np.uint64)
    if kind == "all":  # bits past n_tokens set too: they are not read
        return np.full((t, words), 0xFFFFFFFFFFFFFFFF, np.uint64)
    bits = rng.integers(0, 2 ** 64, (t, words), dtype=np.uint64)
    bits[::3] = 0
    return bits


SHAPES = [  # head_dim, kv heads, heads per kv head, n_past, tokens
    (64, 2, 7, 0, 1), (128, 4, 7, 0, 1), (64, 1, 1, 1, 1), (64, 2, 7, 511, 8), (128, 2, 4, 31, 5),
    (128, 1, 8, 32, 33), (64, 3, 5, 33, 64), (64, 1, 16, 30, 65), (128, 2, 1, 63, 130), (64, 1, 3, 0, 200),
    (128, 4, 7, 1203, 25), (64, 2, 7, 4100, 3),
]


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("kind", ["chain", "tree", "random", "none", "all"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_tree_against_64_bits(hip, stream, cache, kind, shape):
    d, hkv, rep, n_past, t = shape
    rng = np.random.default_rng([d, hkv, rep, n_past, t])
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, make_bits(rng, kind, t))
    run(hip, [s], stream)
    s.check(f"{cache} {kind} {shape}")
    s.close()


@pytest.mark.parametrize("cache", CACHES)
def test_ragged_batch_of_more_than_one_launch(hip, stream, cache):
    rng = np.random.default_rng(5)
    seqs = []
    for i in range(35):
        t = int(rng.integers(1, 20))
        kind = ["chain", "tree", "random"][i % 3]
        n_past = int(rng.choice([0, 1, 40, 333, 1500]))
        seqs.append(Seq(hip, rng, cache, 64, 2, 3, n_past, t, make_bits(rng, kind, t)))
    run(hip, seqs, stream)
    for i, s in enumerate(seqs):
        s.check(f"item {i}")
        s.close()


@pytest.mark.parametrize("cache", ["f32", "f16"])
def test_strides_of_other_layouts(hip, stream, cache):
    # K and V per head (positions inside), queries and outputs with padded heads
    import torch
    rng = np.random.default_rng(6)
    d, hkv, rep, n_past, t = 128, 2, 3, 77, 9
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, make_bits(rng, "tree", t), spare=0)
    s.dk = dev(s.k.transpose(1, 0, 2)).permute(1, 0, 2)
    s.dv = dev(s.v.transpose(1, 0, 2)).permute(1, 0, 2)
    s.src = dict(k=s.dk, v=s.dv)
    qbuf = torch.full((t, hkv * rep + 1, d + 4), 7.0, device="cuda")
    obuf = torch.full((t, hkv * rep + 1, d + 4), -5.0, device="cuda")
    qbuf[:, :-1, :d] = s.dq
    s.dq, s.out = qbuf[:, :-1, :d], obuf[:, :-1, :d]
    run(hip, [s], stream)
    s.check("strided")
    assert torch.all(obuf[:, -1] == -5.0) and torch.all(obuf[:, :, d:] == -5.0)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d", [64, 128])
def test_what_a_query_does_not_see_never_shows(hip, stream, cache, d):
    # infinities and NaN in drafted rows that only some queries see
    rng = np.random.default_rng(7)
    hkv, rep, n_past, t = 2, 3, 45, 40
    n = n_past + t
    k = rng.standard_normal((n + 2, hkv, d)).astype(np.float32)
    v = rng.standard_normal((n + 2, hkv, d)).astype(np.float32)
    bad = [3, 17, 30]
    k[n_past + bad[0]] = np.nan
    v[n_past + bad[1], :, 5] = np.inf
    v[n_past + bad[2], 1] = np.nan
    v[n_past + bad[0], 0, d - 1] = -np.inf
    bits = make_bits(rng, "tree", t)
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, bits, spare=2, k=k, v=v)
    run(hip, [s], stream)
    got = s.out.cpu().numpy()
    seen = ref.visible(n_past, t, bits)
    clean = ~seen[:, [n_past + b for b in bad]].any(1)
    assert clean.sum() >= 5 and (~clean).sum() >= 3
    kk, vv = (np.where(np.isfinite(x), x, 0).astype(np.float64) for x in (s.k, s.v))
    want = ref.attention(s.q, kk, vv, seen, s.scale)
    tol = ref.attention_tolerance(s.q, kk, vv, seen, s.scale)
    assert np.abs(got[clean] - want[clean]).max() <= tol
    # a query that sees them shows it
    assert np.all(np.isnan(got[seen[:, n_past + bad[0]]]))
    sees_inf = seen[:, n_past + bad[1]] & ~seen[:, n_past + bad[0]] & ~seen[:, n_past + bad[2]]
    assert not np.isfinite(got[sees_inf][..., 5]).any()
    if cache != "q8":  # one element of a row does not spread over the row's dims
        assert np.isfinite(got[sees_inf][..., :5]).all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("qmul,kmul,vmul", [(1e4, 1e-3, 1e3), (1e-5, 1e3, 1e-4), (30.0, 1.0, 1.0), (2e30, 1e-30, 1.0)])
def test_magnitudes(hip, stream, cache, qmul, kmul, vmul):
    if cache == "f16" and kmul < 1e-20:
        kmul, qmul = 1e-4, 1e4  # (f16 has no smaller keys)
    if cache == "q8" and kmul < 1e-20:
        kmul, qmul = 1e-3, 2e3
    rng = np.random.default_rng(8)
    d, hkv, rep, n_past, t = 64, 2, 4, 300, 12
    n = n_past + t
    k = (rng.standard_normal((n + 1, hkv, d)) * kmul).astype(np.float32)
    v = (rng.standard_normal((n + 1, hkv, d)) * vmul).astype(np.float32)
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, make_bits(rng, "tree", t), spare=1, qmul=qmul, k=k, v=v)
    run(hip, [s], stream)
    s.check(f"{cache} {qmul} {kmul} {vmul}")
    s.close()


def test_v_rows_of_growing_scale(hip, stream):
    # an 8-bit cache whose V rows grow and shrink by powers of ten from row to row
    rng = np.random.default_rng(9)
    d, hkv, rep, n_past, t = 128, 1, 8, 500, 8
    n = n_past + t
    v = rng.standard_normal((n + 1, hkv, d)) * 10.0 ** rng.integers(-5, 5, (n + 1, hkv, 1))
    k = rng.standard_normal((n + 1, hkv, d)).astype(np.float32)
    s = Seq(hip, rng, "q8", d, hkv, rep, n_past, t, None, spare=1, k=k, v=v.astype(np.float32))
    run(hip, [s], stream)
    s.check("growing")
    s.close()


def test_rows_more_than_32_bits_apart(hip, stream):
    # positions 1 MiB apart: the last rows lie past 4 GiB
    import torch
    rng = np.random.default_rng(10)
    d, n_past, t = 64, 4300, 5
    n = n_past + t
    s = Seq(hip, rng, "f16", d, 1, 2, n_past, t, make_bits(rng, "tree", t), spare=0)
    big = torch.zeros((n, 1 << 19), device="cuda", dtype=torch.float16)
    big[:, :d], big[:, d:2 * d] = s.dk[:, 0], s.dv[:, 0]
    s.src = dict(k=big[:, None, :d], v=big[:, None, d:2 * d])
    run(hip, [s], stream)
    s.check("far rows")


@pytest.mark.parametrize("cache", CACHES)
def test_the_same_bits_every_time_and_on_another_stream(hip, stream, cache):
    import torch
    rng = np.random.default_rng(11)
    s = Seq(hip, rng, cache, 128, 4, 7, 2000, 20, make_bits(rng, "tree", 20))
    run(hip, [s], stream)
    first = s.out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        s.out.fill_(float("nan"))
        torch.cuda.synchronize()
        run(hip, [s], side.cuda_stream)
        assert torch.equal(first, s.out)
    s.close()


@pytest.mark.parametrize("cache", CACHES)
def test_captured_and_replayed(hip, stream, cache):
    # two graphs that share a workspace, replayed in turn with eager calls between
    import torch
    rng = np.random.default_rng(12)
    seqs = [Seq(hip, rng, cache, 64, 2, 7, 1500, 10, make_bits(rng, "tree", 10)),
            Seq(hip, rng, cache, 64, 2, 7, 700, 30, make_bits(rng, "tree", 30))]
    ws = hip.workspace_create(2, 14, 64)
    want = []
    for s in seqs:
        run(hip, [s], stream, ws)
        s.check("eager")
        want.append(s.out.clone())
    side = torch.cuda.Stream()
    graphs = []
    for s in seqs:
        g = torch.cuda.CUDAGraph()
        items = (mh.AttnArgs * 1)(s.args(None, ws))
        masks = mh.tree_masks([s.dbits])
        with torch.cuda.graph(g, stream=side):
            hip.check(hip.mi_hip_attn_tree(items, masks, 1, torch.cuda.current_stream().cuda_stream))
        graphs.append(g)
    for _ in range(4):
        for s, g, w in zip(seqs, graphs, want):
            s.out.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(s.out, w)
        run(hip, [seqs[0]], stream, ws)
        assert torch.equal(seqs[0].out, want[0])
    # a replay reads the mask, queries and cache as they are then
    s = seqs[0]
    s.bits = make_bits(rng, "random", s.t)
    s.dbits.copy_(dev_bits(s.bits))
    graphs[0].replay()
    torch.cuda.synchronize()
    s.check("new mask")
    for s in seqs:
        s.close()
    hip.check(hip.mi_hip_workspace_destroy(ws))


def test_a_small_workspace_limits_the_splits_only(hip, stream):
    # a workspace for 64 dims holds fewer records of 128
    rng = np.random.default_rng(13)
    ws = hip.workspace_create(1, 1, 64)
    s = Seq(hip, rng, "f16", 128, 2, 8, 9000, 16, make_bits(rng, "tree", 16))
    run(hip, [s], stream, ws)
    s.check("small workspace")
    hip.check(hip.mi_hip_workspace_destroy(ws))


def test_decode_launches_after_tree_launches_on_one_workspace(hip, stream):
    # the decode kernels keep stamped records in the workspace: a tree launch leaves them alone
    import torch
    rng = np.random.default_rng(14)
    ws = hip.workspace_create(2, 14, 64)
    s = Seq(hip, rng, "f32", 64, 2, 7, 3000, 1, None)
    want = ref.attention(s.q, s.k, s.v, ref.visible(3000, 1), s.scale)
    for _ in range(3):
        run(hip, [s], stream, ws)
        s.check("tree")
        s.out.fill_(float("nan"))
        a = s.args(stream, ws)
        hip.check(hip.mi_hip_attn_fwd(ctypes.byref(a)))
        torch.cuda.synchronize()
        assert np.abs(s.out.cpu().numpy() - want).max() <= 1e-4
    rc, fallbacks, lost = hip.workspace_check(ws, stream)
    assert rc == 0 and lost == 0
    hip.check(hip.mi_hip_workspace_destroy(ws))


def test_an_8_bit_cache_behind_the_other_entry_points(hip, stream):
    # mi_hip_attn_fwd (one token and a chunk) and mi_hip_attn_decode_batch
    import torch
    rng = np.random.default_rng(15)
    for n_past, t in ((700, 1), (100, 70)):
        s = Seq(hip, rng, "q8", 128, 4, 7, n_past, t, None)
        a = s.args(stream)
        hip.check(hip.mi_hip_attn_fwd(ctypes.byref(a)))
        torch.cuda.synchronize()
        s.check(f"attn_fwd {t}")
        assert hip.mi_hip_attn_fwd_reference_order(ctypes.byref(a)) == 5
        if t == 1:
            assert hip.mi_hip_attn_decode_batch_noalloc(ctypes.byref(a), 1, stream) == 5
            s.out.fill_(float("nan"))
            items = (mh.AttnArgs * 1)(a)
            hip.check(hip.mi_hip_attn_decode_batch(items, 1, stream))
            torch.cuda.synchronize()
            s.check("decode_batch")
        s.close()


def test_no_allocation(hip, stream):
    rng = np.random.default_rng(16)
    s = Seq(hip, rng, "f16", 64, 2, 7, 5000, 12, make_bits(rng, "tree", 12))
    before = hip.alloc_stats()
    run(hip, [s], stream)
    after = hip.alloc_stats()
    assert (after.n_malloc, after.n_free) == (before.n_malloc, before.n_free)
    s.check("no allocation")
