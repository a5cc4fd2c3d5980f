"""The serving operators at the ends of their ranges: values that are not finite in the first keys of
many workgroups, rows of very small values, positions far apart, sources of any alignment, caches and
workspaces under an allocation limit. References in 64 bits."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref
from test_kv8_gpu import dev, tensor_at
from test_tree_gpu import CACHES, Seq, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("d", [64, 128])
def test_marks_of_first_tiles_in_many_workgroups(hip, stream, cache, d):
    # every workgroup's first tile holds V rows that are not finite: queries that see one show it, the others
    # never do, in every workgroup and on every run
    rng = np.random.default_rng([d, 20])
    hkv, rep, t, items = 8, 4, 12, 24
    bits = np.array([[1 << j] for j in range(t)], np.uint64)  # every query sees itself
    seqs = []
    for i in range(items):
        k, v = (rng.standard_normal((t + 1, hkv, d)).astype(np.float32) for _ in range(2))
        v[i % t, :, (7 * i) % d] = np.nan
        v[(i + 5) % t, :, (7 * i + 1) % d] = np.inf
        seqs.append(Seq(hip, rng, cache, d, hkv, rep, 0, t, bits, spare=1, k=k, v=v))
    for _ in range(10):
        for s in seqs:
            s.out.fill_(0.0)
        run(hip, seqs, stream)
        for i, s in enumerate(seqs):
            got = s.out.cpu().numpy()
            want = np.repeat(s.v.astype(np.float64), rep, 1)  # one key: its V row
            bad = ~np.isfinite(want)
            assert np.array_equal(~np.isfinite(got), bad)
            # (a sum of one term: the pairs' 2^-22 of the row's largest and a few roundings)
            assert np.all(np.abs(got - want)[~bad] <= 2.0 ** -21 * np.abs(want[~bad]).max())
    for s in seqs:
        s.close()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rep,t", [(3, 10), (4, 24)])  # 30 rows per KV head, 96
@pytest.mark.parametrize("qmul,kmul", [(1e36, 1e-36), (1e30, 1e-30), (1e-36, 1e36), (1e-30, 1e30)])
def test_small_keys_and_small_queries(hip, stream, d, rep, t, qmul, kmul):
    # an F32 cache: scores of ordinary size from keys or queries at the ends of float's range
    rng = np.random.default_rng([d, rep, t, 21])
    hkv, n_past = 2, 200
    n = n_past + t
    k = (rng.standard_normal((n + 1, hkv, d)) * kmul).astype(np.float32)
    s = Seq(hip, rng, "f32", d, hkv, rep, n_past, t, None, spare=1, qmul=qmul, k=k)
    run(hip, [s], stream)
    s.check(f"{d} {rep} {t} {qmul} {kmul}")
    s.close()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rep,t", [(3, 10), (4, 24)])  # 30 rows per KV head, 96
@pytest.mark.parametrize("vmul", [1e-26, 1e-30, 1e-33, 1e-36])
def test_small_values(hip, stream, d, rep, t, vmul):
    # an F32 cache whose V rows are all small. A query that sees one key gives its V row: at most 2^-21 of the
    # row's largest off (values and probabilities as pairs, 2^-22 each, and a few roundings of 2^-24 that cancel
    # no digits: 2^-20 with them), or 2^-123 (the resolution 2^-124 of values below 2^-102, and the
    # probability's as much)
    rng = np.random.default_rng([d, rep, t, 22])
    hkv, n_past = 2, 33
    n = n_past + t
    v = (rng.standard_normal((n + 1, hkv, d)) * vmul).astype(np.float32)
    s = Seq(hip, rng, "f32", d, hkv, rep, n_past, t, None, spare=1, v=v)
    run(hip, [s], stream)
    got = s.out.cpu().numpy().astype(np.float64)
    seen = ref.visible(n_past, t, None)
    want = ref.attention(s.q, s.k, s.v, seen, s.scale)
    assert np.abs(got - want).max() <= ref.attention_tolerance(s.q, s.k, s.v, seen, s.scale) + 2.0 ** -123
    s.close()
    bits = np.array([[1 << j] for j in range(t)], np.uint64)
    one = Seq(hip, rng, "f32", d, hkv, rep, 0, t, bits, spare=1, v=v[n_past:].copy())
    run(hip, [one], stream)
    want = np.repeat(one.v.astype(np.float64), rep, 1)
    tol = 2.0 ** -20 * np.abs(want).max(-1, keepdims=True) + 2.0 ** -123
    assert np.all(np.abs(one.out.cpu().numpy() - want) <= tol)
    one.close()


@pytest.mark.parametrize("d,hkv,n_dims", [(64, 2, 64), (128, 3, 128), (64, 2, 20), (128, 1, 96)])
@pytest.mark.parametrize("norm", [False, True])
def test_the_8_bit_keys_of_sources_of_any_alignment(hip, stream, d, hkv, n_dims, norm):
    # K's 8-bit form is that of the float nearest to its 64-bit value, however the source's rows lie and
    # whatever part of them is rotated. (The kernels' and the reference's 64-bit values differ by parts in 2^52,
    # which moves a float, and then a whole number, once in far more values than these.)
    import torch
    rng = np.random.default_rng([d, n_dims, norm])
    t = 2000
    k = rng.standard_normal((t, hkv, d)).astype(np.float32) * 3
    w = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
    f = (1e6 ** (-np.arange(0, n_dims, 2, dtype=np.float64) / n_dims)).astype(np.float32)
    want = ref.norm_rope(k, w if norm else None, 1e-6, np.arange(t, dtype=np.int32), f).astype(np.float32)
    want_q, want_scale = ref.quantize(want, 32)
    apart = torch.full((t, hkv, d + 1), 9.0, device="cuda")  # rows that start at any 4 bytes
    apart[:, :, :d] = dev(k)
    dw = dev(w)
    for dk in (dev(k), apart[:, :, :d]):
        kv = hip.kv_create(1, t, hkv, d, hkv, mh.MI_HIP_TYPE_Q8)
        a = mh.norm_rope_args(kv, 0, 0, n_dims, 1e6, stream, dk, dk, freq=f, k_norm=dw if norm else None, eps=1e-6)
        hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
        torch.cuda.synchronize()
        q = tensor_at(hip.kv_view(kv, 0, 0)[0], (t, hkv, d), "|i1").cpu().numpy()
        scale = tensor_at(hip.kv_scales(kv, 0, 0)[0], (t, hkv, d // 32), "<f2").cpu().numpy()
        assert np.array_equal(scale, want_scale)
        assert np.array_equal(q, want_q.reshape(q.shape))
        hip.check(hip.mi_hip_kv_destroy(kv))


@pytest.mark.parametrize("d", [64, 128])
def test_tiles_whose_rows_pass_2_and_4_gib(hip, stream, d):
    # positions 48 MiB apart: with 64 dims a tile of 64 keys is 3 GiB long
    import torch
    rng = np.random.default_rng([d, 23])
    n_past, t, rep = 100, 12, 4
    n = n_past + t
    s = Seq(hip, rng, "f16", d, 1, rep, n_past, t, None, spare=0)
    far = torch.empty((n, 24 << 20), device="cuda", dtype=torch.float16)
    far[:, :d], far[:, d:2 * d] = s.dk[:, 0], s.dv[:, 0]
    s.src = dict(k=far[:, None, :d], v=far[:, None, d:2 * d])
    run(hip, [s], stream)
    s.check("far rows")


def test_caches_and_workspaces_where_a_limit_leaves_no_room_for_the_parts(hip, stream):
    # made without them: attention then keeps every item's keys in one split, greedy ids are refused
    import torch
    rng = np.random.default_rng(24)
    d, hkv, rep, n_past, t = 64, 2, 7, 700, 9
    n = n_past + t
    x = dev(rng.standard_normal((3, 5000)).astype(np.float32))
    out, ids = torch.empty_like(x), torch.empty(3, device="cuda", dtype=torch.int32)
    before = hip.alloc_stats().bytes_live
    kv = hip.kv_create(1, n, hkv, d, hkv * rep, mh.MI_TYPE_F16)
    whole = hip.alloc_stats().bytes_live - before
    hip.check(hip.mi_hip_kv_destroy(kv))
    ws = hip.workspace_create(hkv, hkv * rep, d)
    ws_whole = hip.alloc_stats().bytes_live - before
    hip.check(hip.mi_hip_workspace_destroy(ws))
    try:
        hip.check(hip.mi_hip_set_alloc_limit(before + whole - (1 << 20)))
        kv = hip.kv_create(1, n, hkv, d, hkv * rep, mh.MI_TYPE_F16)
        assert whole - (34 << 20) < hip.alloc_stats().bytes_live - before <= whole - (16 << 20)
        hip.check(hip.mi_hip_set_alloc_limit(hip.alloc_stats().bytes_live + ws_whole - (1 << 20)))
        ws = hip.workspace_create(hkv, hkv * rep, d)
        # and a limit below what they need without parts still refuses
        hip.check(hip.mi_hip_set_alloc_limit(hip.alloc_stats().bytes_live + 1000))
        with pytest.raises(mh.MiHipError) as e:
            hip.workspace_create(hkv, hkv * rep, d)
        assert e.value.code == 4
    finally:
        hip.check(hip.mi_hip_set_alloc_limit(0))
    bits, _ = ref.random_tree(rng, t)
    s = Seq(hip, rng, "f16", d, hkv, rep, n_past, t, bits, spare=0)
    for which, rows in ((0, s.dk), (1, s.dv)):
        hip.kv_write(kv, 0, which, 0, rows.float(), stream)
    s.src = dict(kv=kv, layer=0)
    run(hip, [s], stream)
    s.check("no parts")
    s.out.fill_(float("nan"))
    run(hip, [s], stream, ws)
    s.check("no parts, own workspace")
    # one token by the decode entry point, which needs none
    one = Seq(hip, rng, "f16", d, hkv, rep, n - 1, 1, None, spare=0, k=s.k.astype(np.float32), v=s.v.astype(np.float32))
    a = one.args(stream, ws)
    hip.check(hip.mi_hip_attn_fwd(ctypes.byref(a)))
    torch.cuda.synchronize()
    want = ref.attention(one.q, one.k, one.v, ref.visible(n - 1, 1), one.scale)
    assert np.abs(one.out.cpu().numpy() - want).max() <= 1e-2  # (an F16 cache's bar; conftest's TOL_F16)
    a = mh.logits_args(x, out, stream, ids=ids, ws=ws)
    assert hip.mi_hip_logits_adjust(ctypes.byref(a)) == 5
    a = mh.logits_args(x, out, stream, ws=ws)
    hip.check(hip.mi_hip_logits_adjust(ctypes.byref(a)))
    torch.cuda.synchronize()
    assert torch.equal(x, out)
    hip.check(hip.mi_hip_workspace_destroy(ws))
    hip.check(hip.mi_hip_kv_destroy(kv))
    assert hip.alloc_stats().bytes_live == before
