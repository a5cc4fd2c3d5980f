"""The serving operators where they can go wrong: every attention kernel (up to 16 rows per KV head, up
to 32, more) with values that are not finite or only some queries see, scores out of range, queries that
are not finite, two calls at once, captured steps, the executor hook on an 8-bit cache. References in 64
bits; tolerances as in the operators' own tests."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref
from test_kv8_gpu import dev, read
from test_nodes_gpu import HostGraph
from test_norm_rope_gpu import bound, freqs
from test_tree_gpu import CACHES, Seq, make_bits, run

pytestmark = pytest.mark.gpu

# (heads per KV head, tokens): 15, 30 and 96 rows per KV head
KERNELS = [(3, 5), (3, 10), (4, 24)]


def finite(x):
    return np.where(np.isfinite(x), x, 0).astype(np.float64)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rep,t", KERNELS)
def test_values_that_are_not_finite_in_rows_some_queries_see(hip, stream, cache, d, rep, t):
    rng = np.random.default_rng([d, rep, t])
    hkv, n_past = 2, 141
    n = n_past + t
    k, v = (rng.standard_normal((n + 2, hkv, d)).astype(np.float32) for _ in range(2))
    bits = np.zeros((t, 1), np.uint64)
    for j in range(t):
        bits[j, 0] = 1 << j  # every query sees itself; the last three see one bad row each
    k[n_past] = np.nan
    v[n_past + 1, :, 5] = np.inf
    v[n_past + 2, 1] = np.nan
    v[n_past, 0, d - 1] = -np.inf
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, bits, spare=2, k=k, v=v)
    run(hip, [s], stream)
    got = s.out.cpu().numpy()
    seen = ref.visible(n_past, t, bits)
    want = ref.attention(s.q, finite(s.k), finite(s.v), seen, s.scale)
    tol = ref.attention_tolerance(s.q, finite(s.k), finite(s.v), seen, s.scale)
    assert np.abs(got[3:] - want[3:]).max() <= tol
    assert np.isnan(got[0]).all()
    assert not np.isfinite(got[1][:, 5]).any()
    assert np.isnan(got[2][rep:]).all() and np.abs(got[2][:rep] - want[2][:rep]).max() <= tol
    if cache != "q8":  # one element of a row does not spread over the row's dims
        rest = np.arange(d) != 5
        assert np.abs(got[1][:, rest] - want[1][:, rest]).max() <= tol
    s.close()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rep,t", KERNELS)
def test_huge_rows_that_other_queries_see(hip, stream, cache, d, rep, t):
    # finite K and V rows at the top of the type's range, each seen by one query only: the others keep
    # their precision
    rng = np.random.default_rng([d, rep, t, 1])
    hkv, n_past = 2, 70
    n = n_past + t
    big = {"f32": 3e37, "f16": 6e4, "q8": 8e6}[cache]
    k, v = (rng.standard_normal((n + 2, hkv, d)).astype(np.float32) for _ in range(2))
    k[n_past + 1] *= big / np.abs(k[n_past + 1]).max()
    v[n_past + 2] *= big / np.abs(v[n_past + 2]).max()
    bits = np.array([[1 << j] for j in range(t)], np.uint64)
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, bits, spare=2, k=k, v=v, qmul=0.2)
    run(hip, [s], stream)
    got = s.out.cpu().numpy()
    seen = ref.visible(n_past, t, bits)
    rows = [0] + list(range(3, t))  # (rows 1 and 2 see the huge ones)
    want = ref.attention(s.q[rows], s.k, s.v, seen[rows], s.scale)
    tol = ref.attention_tolerance(s.q[rows], s.k, s.v, seen[rows], s.scale)
    assert np.abs(got[rows] - want).max() <= tol
    want = ref.attention(s.q[2:3], s.k, s.v, seen[2:3], s.scale)
    assert np.abs(got[2:3] - want).max() <= ref.attention_tolerance(s.q[2:3], s.k, s.v, seen[2:3], s.scale)
    s.close()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rep,t", KERNELS)
def test_rows_of_very_different_sizes(hip, stream, cache, d, rep, t):
    # K and V rows that grow and shrink by powers of ten from row to row; per element within the tolerance of
    # the largest V row that the query sees
    rng = np.random.default_rng([d, rep, t, 4])
    hkv, n_past = 2, 400
    n = n_past + t
    lo, hi = {"f32": (-12, 12), "f16": (-3, 4), "q8": (-5, 6)}[cache]
    k = rng.standard_normal((n + 1, hkv, d)) * 10.0 ** rng.integers(-3, 1, (n + 1, hkv, 1))
    v = rng.standard_normal((n + 1, hkv, d)) * 10.0 ** rng.integers(lo, hi, (n + 1, hkv, 1))
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, None, spare=1, k=k.astype(np.float32), v=v.astype(np.float32))
    run(hip, [s], stream)
    s.check(f"{cache} {d} {rep} {t}")
    s.close()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("rep,t", KERNELS)
def test_queries_that_are_not_finite_and_scores_below_the_range(hip, stream, cache, rep, t):
    rng = np.random.default_rng([rep, t, 2])
    d, hkv, n_past = 64, 2, 100
    k = np.abs(rng.standard_normal((n_past + t + 1, hkv, d))).astype(np.float32) + 1.0
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, None, spare=1, k=k)
    s.q[1, 0] = np.nan
    s.q[2, rep, 3] = np.inf
    s.q[3, :] = -3e38  # every score is below float's range
    s.dq.copy_(dev(s.q))
    run(hip, [s], stream)
    got = s.out.cpu().numpy()
    assert np.isnan(got[1, 0]).all() and np.isnan(got[2, rep]).all()
    assert np.all(got[3] == 0.0)
    good = np.ones((t, hkv * rep), bool)
    good[1, 0] = good[2, rep] = False
    good[3] = False
    seen = ref.visible(n_past, t)
    q = np.where(good[..., None], s.q, 0)
    want = ref.attention(q, s.k, s.v, seen, s.scale)
    assert np.abs(got[good] - want[good]).max() <= ref.attention_tolerance(q, s.k, s.v, seen, s.scale)
    s.close()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d,hkv,rep,n_past,t", [(64, 1, 16, 2047, 1), (64, 1, 17, 2047, 1), (128, 1, 32, 900, 1),
                                                (128, 2, 33, 900, 1), (64, 1, 40, 31, 1), (128, 5, 1, 6000, 16),
                                                (128, 1, 3, 0, 11)])
def test_groups_at_the_borders_between_the_kernels(hip, stream, cache, d, hkv, rep, n_past, t):
    rng = np.random.default_rng([d, hkv, rep, n_past, t])
    s = Seq(hip, rng, cache, d, hkv, rep, n_past, t, make_bits(rng, "tree", t))
    run(hip, [s], stream)
    s.check(f"{cache} {d} {hkv} {rep} {n_past} {t}")
    s.close()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d,hkv,rep,items", [  # n_past, tokens and mask of each item
    (64, 1, 7, [(0, 500, "chain")]), (64, 1, 7, [(900, 300, "random")]), (128, 4, 7, [(70, 260, "chain")]),
    (128, 3, 5, [(0, 300, "chain"), (1000, 1, "chain"), (33, 90, "tree"), (5, 450, "chain"), (2000, 40, "random")]),
    (64, 2, 7, [(1500, 400, "chain"), (0, 130, "all"), (257, 19, "chain")])])
def test_many_row_tiles_and_mixed_batches(hip, stream, cache, d, hkv, rep, items):
    # row tiles that cut their own keys, dealt in parts where a call has few (KV head, split) units
    rng = np.random.default_rng([d, hkv, rep, len(items)])
    seqs = [Seq(hip, rng, cache, d, hkv, rep, n_past, t, make_bits(rng, kind, t)) for n_past, t, kind in items]
    run(hip, seqs, stream)
    for i, s in enumerate(seqs):
        s.check(f"item {i} {items[i]}")
        s.close()


def test_two_calls_at_once_on_their_own_workspaces(hip, stream):
    import torch
    rng = np.random.default_rng(3)
    seqs = [Seq(hip, rng, "f16", 128, 4, 7, 6000, 25, make_bits(rng, "tree", 25)),
            Seq(hip, rng, "q8", 64, 2, 7, 9000, 8, None)]
    ws = [hip.workspace_create(4, 28, 128), None]  # (the 8-bit cache has its own)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, w, st in zip(seqs, ws, streams):
            items = (mh.AttnArgs * 1)(s.args(st.cuda_stream, w))
            masks = mh.tree_masks([s.dbits])
            hip.check(hip.mi_hip_attn_tree(items, masks, 1, st.cuda_stream))
    torch.cuda.synchronize()
    for s in seqs:
        s.check("at once")
        s.close()
    hip.check(hip.mi_hip_workspace_destroy(ws[0]))


def test_ids_of_two_calls_at_once_on_their_own_workspaces(hip, stream):
    import torch
    rng = np.random.default_rng(7)
    ws = [hip.workspace_create(1, 1, 64) for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    xs = [dev(rng.standard_normal(s).astype(np.float32)) for s in ((3, 151936), (40, 33000))]
    outs = [torch.empty_like(x) for x in xs]
    ids = [torch.full((20, len(x)), -5, device="cuda", dtype=torch.int32) for x in xs]
    torch.cuda.synchronize()
    for i in range(20):
        for x, out, d, w, st in zip(xs, outs, ids, ws, streams):
            a = mh.logits_args(x, out, st.cuda_stream, ids=d[i])
            a.ws = w
            hip.check(hip.mi_hip_logits_adjust(ctypes.byref(a)))
    torch.cuda.synchronize()
    for x, d in zip(xs, ids):
        assert torch.equal(d, x.argmax(1).to(torch.int32).expand(20, -1))
    for w in ws:
        hip.check(hip.mi_hip_workspace_destroy(w))


@pytest.mark.parametrize("kind", [mh.MI_TYPE_F32, mh.MI_TYPE_F16, mh.MI_HIP_TYPE_Q8])
def test_a_captured_step_replays(hip, stream, kind):
    # norms and RoPE with append, attention, the kept rows and a read back in one graph, replayed with
    # eager calls and other tokens between: every replay gives the eager bits
    import torch
    rng = np.random.default_rng(4)
    d, hkv, rep, n_past, t = 64, 2, 7, 700, 12
    h = hkv * rep
    bits, depth = ref.random_tree(rng, t)
    dbits, pos = dev(bits.view(np.int64)), dev((n_past + depth).astype(np.int32))
    w = dev((1 + 0.1 * rng.standard_normal(d)).astype(np.float32))
    kv = hip.kv_create(2, n_past + t, hkv, d, h, kind)
    for layer in range(2):
        for which in range(2):
            hip.kv_write(kv, layer, which, 0, dev(rng.standard_normal((n_past + t, hkv, d)).astype(np.float32)), None)
    q, k, v = (torch.empty((t, n, d), device="cuda") for n in (h, hkv, hkv))
    qr, out, back = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k)
    keep = np.array([0, 2, 5, 9])

    def step(st):
        a = mh.norm_rope_args(kv, 1, n_past, d, 1e6, st, k, v, q=q, q_out=qr, pos=pos, q_norm=w, k_norm=w, eps=1e-6)
        hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
        items = (mh.AttnArgs * 1)(mh.attn_args(qr, out, rep, n_past, 0.125, st, kv=kv, layer=1))
        masks = mh.tree_masks([dbits])
        hip.check(hip.mi_hip_attn_tree(items, masks, 1, st))
        hip.kv_keep(kv, n_past, keep, st)
        hip.kv_read(kv, 1, 0, n_past, back, st)

    def tokens():
        for x in (q, k, v):
            x.copy_(dev(rng.standard_normal(tuple(x.shape)).astype(np.float32)))

    tokens()
    step(stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        step(torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        tokens()
        step(stream)
        torch.cuda.synchronize()
        want = [x.clone() for x in (qr, out, back)]
        for x in (qr, out, back):
            x.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip((qr, out, back), want):
            assert torch.equal(x, y)
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_the_executor_hook_on_an_8_bit_cache(hip):
    d, h, hkv, n_ctx = 64, 14, 2, 128
    rng = np.random.default_rng(5)
    q = rng.standard_normal((n_ctx, h, d)).astype(np.float32)
    k, v = (rng.standard_normal((n_ctx, hkv, d)).astype(np.float32) for _ in range(2))
    kq, vq = ref.q8(k, 0), ref.q8(v, 1)
    kv = hip.kv_create(2, n_ctx, hkv, d, h, mh.MI_HIP_TYPE_Q8)
    hg = HostGraph(hip, kv, 1, d, h, hkv, n_ctx)
    for n_past, t in ((0, 50), (50, 1), (51, 1), (52, 9)):
        rows = slice(n_past, n_past + t)
        hg.build(q[rows], k[rows], v[rows], n_past, 0.125)
        out = hg.run(nth=2)
        seen = ref.visible(n_past, t)
        ks, vs = kq[:n_past + t], vq[:n_past + t]
        want = ref.attention(q[rows], ks, vs, seen, 0.125)
        assert np.abs(out - want).max() <= ref.attention_tolerance(q[rows], ks, vs, seen, 0.125)
    hip.check(hip.mi_hip_kv_destroy(kv))


@pytest.mark.parametrize("n_dims", [64, 20])  # the form for whole rows, the form for any
@pytest.mark.parametrize("kind", [mh.MI_TYPE_F32, mh.MI_HIP_TYPE_Q8])
def test_norms_of_rows_whose_squares_leave_the_range(hip, stream, n_dims, kind):
    import torch
    rng = np.random.default_rng(6)
    d, hkv, h = 64, 2, 4
    mags = np.array([1e25, 1e-25, 3e36, 1e-36, 1.0], np.float32)
    t = len(mags)
    q, k = (rng.standard_normal((t, n, d)).astype(np.float32) * mags[:, None, None] for n in (h, hkv))
    v = rng.standard_normal((t, hkv, d)).astype(np.float32)
    w, f = (1 + 0.1 * rng.standard_normal(d)).astype(np.float32), freqs(n_dims)
    kv = hip.kv_create(1, t, hkv, d, h, kind)
    out = torch.full((t, h, d), float("nan"), device="cuda")
    dw, dq, dk, dv = dev(w), dev(q), dev(k), dev(v)
    a = mh.norm_rope_args(kv, 0, 0, n_dims, 1e6, stream, dk, dv, q=dq, q_out=out, freq=f, q_norm=dw, k_norm=dw, eps=0.0)
    hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    pos = np.arange(t, dtype=np.int32)
    want = ref.norm_rope(q, w, 0.0, pos, f)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound(want, d))
    want = ref.norm_rope(k, w, 0.0, pos, f)
    got = read(hip, kv, 0, 0, 0, t, hkv, d, stream)
    step = 0.0 if kind == mh.MI_TYPE_F32 else \
        np.repeat(ref.quantize(want.astype(np.float32), 32)[1], 32, -1) * (0.5 + 2.0 ** -10 * 127)
    assert np.all(np.abs(got - want) <= bound(want, d) + step)
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_queries_in_place_need_the_same_strides(hip, stream):
    import torch
    for kind in (mh.MI_TYPE_F16, mh.MI_HIP_TYPE_Q8):
        kv = hip.kv_create(1, 4, 2, 64, 4, kind)
        x, k = torch.zeros((4, 8, 64), device="cuda"), torch.zeros((4, 2, 64), device="cuda")
        a = mh.norm_rope_args(kv, 0, 0, 64, 1e6, stream, k, k, q=x[:, :4], q_out=x[:, :4])
        assert hip.mi_hip_norm_rope_append(ctypes.byref(a)) == 0
        a = mh.norm_rope_args(kv, 0, 0, 64, 1e6, stream, k, k, q=x[:, :4], q_out=x[:, ::2])
        assert hip.mi_hip_norm_rope_append(ctypes.byref(a)) == 1
        a.n_head = 2
        assert hip.mi_hip_norm_rope_append(ctypes.byref(a)) == 1
        torch.cuda.synchronize()
        hip.check(hip.mi_hip_kv_destroy(kv))
