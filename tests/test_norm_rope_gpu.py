"""Norms of queries and keys per head, rotation and append (mi_hip_norm_rope_append) against 64 bits.

Tolerance, with e = 2^-24 and y the 64-bit result of the norm: the sum of squares of d terms is at
most d e off relative, its root half of that, and the root, the quotient and the two products add four
roundings; the rotation's cosine, sine, two products and sum add at most four more of the pair's
norm. So an element is at most (d / 2 + 8) e off relative to the largest element of its row times
sqrt(2). An F16 cache adds half a step (2^-11 of the value, at least 2^-25). An 8-bit cache may round
such a value to the other neighbour: it is at most d / 2 plus that error away from the 64-bit value."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref
from test_kv8_gpu import dev, read

pytestmark = pytest.mark.gpu

KINDS = {"f32": mh.MI_TYPE_F32, "f16": mh.MI_TYPE_F16, "q8": mh.MI_HIP_TYPE_Q8}
EPS = 1e-6


def freqs(n_dims, base=1e6):
    return (base ** (-np.arange(0, n_dims, 2, dtype=np.float64) / max(n_dims, 1))).astype(np.float32)


def bound(want, d):
    return (d / 2 + 8) * 2.0 ** -24 * np.sqrt(2) * np.abs(want).max(-1, keepdims=True) + 1e-37


def check_cache(got, want, tol, cache, which):
    if cache == "f32":
        lim = tol
    elif cache == "f16":
        lim = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    else:
        step = ref.quantize(want.astype(np.float32), 32 if which == 0 else want.shape[-1])[1]
        step = np.repeat(step, want.shape[-1] // step.shape[-1], -1)
        # (the scale itself may be the next f16 number where its border lies within the error)
        lim = tol + step * (0.5 + 2.0 ** -10 * 127)
    assert np.all(np.abs(got - want) <= lim), np.max(np.abs(got - want) - lim)


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("d,hkv,rep,t,n_past,n_dims,norm,positions", [
    (64, 2, 7, 1, 600, 64, "qk", None), (128, 4, 7, 25, 2000, 128, "qk", "tree"), (64, 2, 7, 33, 0, 64, "", None),
    (128, 1, 1, 5, 3, 128, "q", "far"), (64, 3, 2, 70, 10, 32, "k", "tree"), (128, 2, 3, 9, 1, 0, "qk", None),
    (128, 2, 4, 300, 17, 96, "qk", None), (64, 1, 16, 2, 5, 2, "", "far"),
])
def test_against_64_bits(hip, stream, cache, d, hkv, rep, t, n_past, n_dims, norm, positions):
    import torch
    rng = np.random.default_rng([d, hkv, t, n_dims])
    h = hkv * rep
    q, k, v = (rng.standard_normal((t, n, d)).astype(np.float32) * 3 for n in (h, hkv, hkv))
    wq, wk = ((1 + 0.3 * rng.standard_normal(d)).astype(np.float32) for _ in range(2))
    pos = n_past + np.arange(t, dtype=np.int32)
    if positions == "tree":
        pos = (n_past + ref.random_tree(rng, t)[1]).astype(np.int32)
    elif positions == "far":
        pos = rng.integers(0, 1 << 20, t).astype(np.int32)
    f = freqs(n_dims)
    kv = hip.kv_create(2, n_past + t + 1, hkv, d, h, KINDS[cache])
    out = torch.full((t, h, d), float("nan"), device="cuda")
    dpos, dwq, dwk = dev(pos), dev(wq), dev(wk)
    dq, dk, dv = dev(q), dev(k), dev(v)
    a = mh.norm_rope_args(kv, 1, n_past, n_dims, 1e6, stream, dk, dv, q=dq, q_out=out,
                          pos=dpos if positions else None, freq=f, q_norm=dwq if "q" in norm else None,
                          k_norm=dwk if "k" in norm else None, eps=EPS)
    hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    want = ref.norm_rope(q, wq if "q" in norm else None, EPS, pos, f)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound(want, d))
    assert np.array_equal(dq.cpu().numpy(), q)
    for which, x in ((0, ref.norm_rope(k, wk if "k" in norm else None, EPS, pos, f)), (1, v.astype(np.float64))):
        got = read(hip, kv, 1, which, 0, n_past + t + 1, hkv, d, stream)
        assert not got[:n_past].any() and not got[n_past + t:].any()  # rows around
        check_cache(got[n_past:n_past + t], x, bound(x, d) if which == 0 else 0 * x, cache, which)
        assert not read(hip, kv, 0, which, 0, n_past + t + 1, hkv, d, stream).any()
    if cache == "q8":  # V is quantised from its own values: exact
        assert np.array_equal(read(hip, kv, 1, 1, n_past, t, hkv, d, stream), ref.q8(v, 1))
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_rows_of_zeros_and_of_large_values(hip, stream):
    import torch
    d, hkv, h, t = 64, 1, 2, 4
    q = np.zeros((t, h, d), np.float32)
    q[1], q[2] = 1e18, 1e-18
    k, v = np.zeros((t, hkv, d), np.float32), np.zeros((t, hkv, d), np.float32)
    w = np.ones(d, np.float32)
    kv = hip.kv_create(1, t, hkv, d, h, mh.MI_HIP_TYPE_Q8)
    out = torch.full((t, h, d), float("nan"), device="cuda")
    dw, dq, dk, dv = dev(w), dev(q), dev(k), dev(v)
    a = mh.norm_rope_args(kv, 0, 0, d, 1e4, stream, dk, dv, q=dq, q_out=out, q_norm=dw, k_norm=dw, eps=EPS)
    hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    f = np.array([np.float32(np.float32(1e4) ** np.float32(-2.0 * p / d)) for p in range(d // 2)], np.float32)
    want = ref.norm_rope(q, w, EPS, np.arange(t, dtype=np.int32), f)
    # (the library's own frequencies are the host's powf values, here numpy's: a step apart at most)
    assert np.all(got[0] == 0) and np.all(got[3] == 0)
    assert np.all(np.abs(got - want) <= bound(want, d) + 4 * 2.0 ** -23 * np.abs(want).max(-1, keepdims=True))
    assert not read(hip, kv, 0, 0, 0, t, hkv, d, stream).any()
    hip.check(hip.mi_hip_kv_destroy(kv))


@pytest.mark.parametrize("n_dims", [64, 20])
@pytest.mark.parametrize("kind", [mh.MI_TYPE_F32, mh.MI_TYPE_F16])
def test_without_norms_the_results_of_rope_append(hip, stream, kind, n_dims):
    import torch
    rng = np.random.default_rng(3)
    d, hkv, h, t, n_past = 64, 2, 14, 19, 13
    dq, dk, dv = (dev(rng.standard_normal((t, n, d)).astype(np.float32)) for n in (h, hkv, hkv))
    res = []
    for fn, make in ((hip.mi_hip_rope_append, mh.rope_args), (hip.mi_hip_norm_rope_append, mh.norm_rope_args)):
        kv = hip.kv_create(1, n_past + t, hkv, d, h, kind)
        out = torch.empty_like(dq)
        a = make(kv, 0, n_past, n_dims, 1e6, stream, dk, dv, q=dq, q_out=out)
        hip.check(fn(ctypes.byref(a)))
        torch.cuda.synchronize()
        res.append([out.cpu().numpy()] + [read(hip, kv, 0, w, 0, n_past + t, hkv, d, stream) for w in (0, 1)])
        hip.check(hip.mi_hip_kv_destroy(kv))
    for x, y in zip(*res):
        assert np.array_equal(x, y)


def test_rope_append_takes_an_8_bit_cache(hip, stream):
    import torch
    rng = np.random.default_rng(4)
    d, hkv, h, t, n_past = 128, 2, 8, 6, 40
    q, k, v = (rng.standard_normal((t, n, d)).astype(np.float32) for n in (h, hkv, hkv))
    dq, dk, dv = dev(q), dev(k), dev(v)
    kv = hip.kv_create(1, n_past + t, hkv, d, h, mh.MI_HIP_TYPE_Q8)
    a = mh.rope_args(kv, 0, n_past, d, 1e6, stream, dk, dv, q=dq)  # in place
    hip.check(hip.mi_hip_rope_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    f32 = hip.kv_create(1, n_past + t, hkv, d, h, mh.MI_TYPE_F32)
    dq2 = dev(q)
    b = mh.rope_args(f32, 0, n_past, d, 1e6, stream, dk, dv, q=dq2)
    hip.check(hip.mi_hip_rope_append(ctypes.byref(b)))
    torch.cuda.synchronize()
    assert torch.equal(dq, dq2)
    rotated = read(hip, f32, 0, 0, n_past, t, hkv, d, stream)
    check_cache(read(hip, kv, 0, 0, n_past, t, hkv, d, stream), rotated.astype(np.float64), bound(rotated, d), "q8", 0)
    assert np.array_equal(read(hip, kv, 0, 1, n_past, t, hkv, d, stream), ref.q8(v, 1))
    for x in (kv, f32):
        hip.check(hip.mi_hip_kv_destroy(x))


@pytest.mark.parametrize("cache", list(KINDS))
def test_strides_and_no_queries(hip, stream, cache):
    # rows padded by an odd number of floats, dims two apart, in place; then K and V alone
    import torch
    rng = np.random.default_rng(5)
    d, hkv, h, t = 128, 2, 6, 11
    q, k, v = (rng.standard_normal((t, n, d)).astype(np.float32) for n in (h, hkv, hkv))
    w = (1 + 0.1 * rng.standard_normal(d)).astype(np.float32)
    f, pos = freqs(d), np.arange(t, dtype=np.int32)
    qb = torch.full((t, h, d + 3), 9.0, device="cuda")
    qb[:, :, :d] = dev(q)
    kb = torch.full((t, hkv, 2 * d), 9.0, device="cuda")
    kb[:, :, ::2] = dev(k)
    vb = dev(v.transpose(1, 0, 2)).permute(1, 0, 2)
    dw = dev(w)
    kv = hip.kv_create(1, t, hkv, d, h, KINDS[cache])
    a = mh.norm_rope_args(kv, 0, 0, d, 1e6, stream, kb[:, :, ::2], vb, q=qb[:, :, :d], freq=f, q_norm=dw, k_norm=dw,
                          eps=EPS)
    hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    want = ref.norm_rope(q, w, EPS, pos, f)
    assert np.all(np.abs(qb[:, :, :d].cpu().numpy() - want) <= bound(want, d)) and torch.all(qb[:, :, d:] == 9.0)
    first = [read(hip, kv, 0, x, 0, t, hkv, d, stream) for x in (0, 1)]
    wk = ref.norm_rope(k, w, EPS, pos, f)
    check_cache(first[0], wk, bound(wk, d), cache, 0)
    check_cache(first[1], v.astype(np.float64), 0 * v, cache, 1)
    dk, dv = dev(k), dev(v)
    a = mh.norm_rope_args(kv, 0, 0, d, 1e6, stream, dk, dv, freq=f, k_norm=dw, eps=EPS)
    hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    check_cache(read(hip, kv, 0, 0, 0, t, hkv, d, stream), wk, bound(wk, d), cache, 0)
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_refusals(hip, stream):
    kv = hip.kv_create(1, 8, 2, 64, 4, mh.MI_HIP_TYPE_Q8)
    import torch
    x = torch.zeros((8, 4, 64), device="cuda")

    def rc(**kw):
        a = mh.norm_rope_args(kv, 0, 0, 64, 1e6, stream, x[:2, :2], x[:2, :2], q=x[:2])
        for n, val in kw.items():
            if n.endswith("_nb"):
                getattr(a, n)[:] = val
            else:
                setattr(a, n, val)
        return hip.mi_hip_norm_rope_append(ctypes.byref(a))
    assert rc() == 0
    assert hip.mi_hip_norm_rope_append(None) == 1
    for kw, code in [(dict(layer=1), 1), (dict(n_past=7), 1), (dict(n_tokens=-1), 1), (dict(n_dims=63), 5),
                     (dict(n_dims=66), 5), (dict(kv=None), 1), (dict(q_out=None), 1), (dict(n_head=3), 1),
                     (dict(n_head=0), 1), (dict(k_nb=(4, 6, 8)), 1), (dict(k=None), 1),
                     (dict(k_norm=x.data_ptr(), eps=float("nan")), 1), (dict(k_norm=x.data_ptr(), eps=-1.0), 1),
                     (dict(pos=x.data_ptr() + 2), 1), (dict(n_past=2 ** 31 - 1, n_tokens=2 ** 31 - 1), 1)]:
        assert rc(**kw) == code, kw
    assert rc(n_tokens=0) == 0
    torch.cuda.synchronize()
    hip.check(hip.mi_hip_kv_destroy(kv))
