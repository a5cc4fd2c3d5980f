"""Rotation by several axes and the append to a paged cache (mi_hip_paged_append) against 64 bits, and
against mi_hip_norm_rope_append bit for bit. Tolerances: test_norm_rope_gpu.py derives them."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as sref
from test_kv8_gpu import dev, read
from test_norm_rope_gpu import EPS, KINDS, bound, check_cache, freqs

pytestmark = pytest.mark.gpu


def rotate(x, w, pos, axis, freq):
    """Rows normed, pair j turned by float(pos[axis[j]] * freq[j]); 64 bits otherwise."""
    y = sref.norm_rope(x, w, EPS, np.zeros(len(x), np.int32), freq)  # (angles of 0: the norm alone)
    half = len(freq)
    p = np.stack([pos[a] for a in axis], 1).astype(np.float32) if half else np.zeros((len(x), 0), np.float32)
    theta = (p * freq[None, :]).astype(np.float32).astype(np.float64)[:, None, :]
    a, b = y[..., :half].copy(), y[..., half:2 * half].copy()
    y[..., :half] = a * np.cos(theta) - b * np.sin(theta)
    y[..., half:2 * half] = a * np.sin(theta) + b * np.cos(theta)
    return y


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("d,hkv,rep,t,page,n_dims,norm,axes,layout", [
    (64, 2, 7, 1, 16, 64, "qk", 1, "one"), (128, 4, 7, 70, 32, 128, "", 3, "sections"), (128, 2, 3, 9, 16, 128, "qk", 3, "turns"),
    (64, 1, 1, 300, 64, 64, "k", 2, "turns"), (64, 3, 2, 33, 16, 32, "q", 4, "random"), (128, 1, 16, 5, 128, 0, "qk", 2, "one"),
    (128, 2, 4, 2500, 256, 128, "qk", 3, "sections"), (128, 2, 2, 40, 16, 96, "", 4, "turns"),
])
def test_against_64_bits(hip, stream, cache, d, hkv, rep, t, page, n_dims, norm, axes, layout):
    import torch
    rng = np.random.default_rng([d, hkv, t, n_dims, axes])
    h, pairs = hkv * rep, n_dims // 2
    q, k, v = (rng.standard_normal((t, n, d)).astype(np.float32) * 3 for n in (h, hkv, hkv))
    wq, wk = ((1 + 0.3 * rng.standard_normal(d)).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, 1 << 17, (axes, t)).astype(np.int32)
    pos[:, 0] = 0
    axis = dict(one=[0] * pairs, sections=[i * axes // max(pairs, 1) for i in range(pairs)], turns=[i % axes for i in range(pairs)],
                random=rng.integers(0, axes, pairs).tolist())[layout]
    f = freqs(n_dims)
    n_pages = -(-t // page) + 2
    slots = rng.permutation(n_pages * page)[:t].astype(np.int32)
    out_of_it = rng.random(t) < 0.2 if t > 4 else np.zeros(t, bool)
    slots[out_of_it] = rng.choice([-1, n_pages * page, 2 ** 31 - 1, -2 ** 31], out_of_it.sum())
    kv = hip.kv_create_paged(2, n_pages, page, hkv, d, h, KINDS[cache])
    out = torch.full((t, h, d), float("nan"), device="cuda")
    wide = torch.full((axes, t + 5), 1 << 30, dtype=torch.int32, device="cuda")  # rows further apart
    wide[:, :t] = dev(pos)
    dslots, dwq, dwk, dq, dk, dv = dev(slots), dev(wq), dev(wk), dev(q), dev(k), dev(v)
    a = mh.paged_append_args(kv, 1, n_dims, 1e6, stream, dk, dv, dslots, wide[:, :t], q=dq, q_out=out,
                             axis=None if layout == "one" else axis, freq=f, q_norm=dwq if "q" in norm else None,
                             k_norm=dwk if "k" in norm else None, eps=EPS)
    hip.check(hip.mi_hip_paged_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    want = rotate(q, wq if "q" in norm else None, pos, axis, f)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound(want, d))
    stored = ~out_of_it
    for which, x in ((0, rotate(k, wk if "k" in norm else None, pos, axis, f)), (1, v.astype(np.float64))):
        got = read(hip, kv, 1, which, 0, n_pages * page, hkv, d, stream)
        rest = np.ones(n_pages * page, bool)
        rest[slots[stored]] = False
        assert not got[rest].any()
        check_cache(got[slots[stored]], x[stored], (bound(x, d) if which == 0 else 0 * x)[stored], cache, which)
        assert not read(hip, kv, 0, which, 0, n_pages * page, hkv, d, stream).any()
    hip.check(hip.mi_hip_kv_destroy(kv))


@pytest.mark.parametrize("cache", list(KINDS))
@pytest.mark.parametrize("d,t,n_dims,strided", [(64, 5, 64, False), (128, 40, 128, False), (128, 3000, 128, False), (64, 30, 64, True),
                                                (128, 11, 64, False)])
def test_one_axis_is_norm_rope_append(hip, stream, cache, d, t, n_dims, strided):
    """The same values, so the same bits, row by row, whatever their order in memory."""
    import torch
    rng = np.random.default_rng([d, t])
    hkv, h, page = 2, 6, 16
    n_pages = -(-t // page)
    perm = rng.permutation(n_pages * page)[:t]
    pos = rng.integers(0, 1 << 16, t).astype(np.int32)
    pad = 2 if strided else 0  # (rows that start at any 4 bytes take the other kernel)
    dq, dk, dv = (dev(rng.standard_normal((t, n, d + pad)).astype(np.float32))[..., :d] for n in (h, hkv, hkv))
    w = dev((1 + 0.3 * rng.standard_normal(d)).astype(np.float32))
    dpos, dslots, f = dev(pos), dev(perm.astype(np.int32)), freqs(n_dims)
    one = hip.kv_create(1, n_pages * page, hkv, d, h, KINDS[cache])
    many = hip.kv_create_paged(1, n_pages, page, hkv, d, h, KINDS[cache])
    outs = [torch.empty((t, h, d), device="cuda") for _ in range(2)]
    a = mh.norm_rope_args(one, 0, 0, n_dims, 1e6, stream, dk, dv, q=dq, q_out=outs[0], pos=dpos, freq=f, q_norm=w, k_norm=w, eps=EPS)
    hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
    b = mh.paged_append_args(many, 0, n_dims, 1e6, stream, dk, dv, dslots, dpos, q=dq, q_out=outs[1], freq=f, q_norm=w, k_norm=w,
                             eps=EPS)
    hip.check(hip.mi_hip_paged_append(ctypes.byref(b)))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
    for which in (0, 1):
        x, y = (read(hip, kv, 0, which, 0, n_pages * page, hkv, d, stream) for kv in (one, many))
        assert np.array_equal(x[:t], y[perm])
    hip.check(hip.mi_hip_kv_destroy(one))
    hip.check(hip.mi_hip_kv_destroy(many))


def test_no_queries_in_place_and_no_tokens(hip, stream):
    import torch
    rng = np.random.default_rng(2)
    d, hkv, h, t, page = 64, 2, 4, 6, 16
    q, k, v = (dev(rng.standard_normal((t, n, d)).astype(np.float32)) for n in (h, hkv, hkv))
    slots, pos = dev(np.arange(t, dtype=np.int32)), dev(np.arange(t, dtype=np.int32) + 100)
    kv = hip.kv_create_paged(1, 2, page, hkv, d, h, mh.MI_TYPE_F32)
    apart = torch.empty_like(q)
    for kw in (dict(q=q, q_out=apart), dict(q=q), dict()):  # elsewhere, in place, none
        a = mh.paged_append_args(kv, 0, d, 1e4, stream, k, v, slots, pos, **kw)
        hip.check(hip.mi_hip_paged_append(ctypes.byref(a)))
    torch.cuda.synchronize()
    assert torch.equal(q, apart)
    before = read(hip, kv, 0, 0, 0, 2 * page, hkv, d, stream)
    a.n_tokens = 0
    hip.check(hip.mi_hip_paged_append(ctypes.byref(a)))
    assert np.array_equal(before, read(hip, kv, 0, 0, 0, 2 * page, hkv, d, stream))
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_refusals(hip, stream):
    import torch
    t, d = 4, 64
    x, i = torch.zeros((t, 2, d), device="cuda"), torch.zeros((2, t), dtype=torch.int32, device="cuda")
    paged = hip.kv_create_paged(2, 3, 16, 2, d, 4, mh.MI_TYPE_F16)
    plain = hip.kv_create(2, 48, 2, d, 4, mh.MI_TYPE_F16)

    def rc(kv, **kw):
        a = mh.paged_append_args(kv, 0, d, 1e4, stream, x, x, i[0], i, axis=[0] * 32)
        for n, v in kw.items():
            if n == "axis5":
                a.axis[5] = v
            else:
                setattr(a, n, v)
        return hip.mi_hip_paged_append(ctypes.byref(a))
    assert rc(paged) == 0
    assert rc(plain) == 5 and "paged" in hip.last_error()
    for kw, code in ((dict(layer=2), 1), (dict(layer=-1), 1), (dict(n_tokens=-1), 1), (dict(n_axes=0), 5), (dict(n_axes=5), 5),
                     (dict(pos_nb=12), 1), (dict(pos_nb=18), 1), (dict(axis5=2), 1), (dict(axis5=-1), 1), (dict(n_dims=66), 5),
                     (dict(n_dims=7), 5), (dict(slots=None), 1), (dict(pos=None), 1), (dict(slots=i.data_ptr() + 2), 1)):
        assert rc(paged, **kw) == code, (kw, hip.last_error())
    # a paged cache is no single sequence's
    q = torch.zeros((1, 4, d), device="cuda")
    args = mh.attn_args(q, q.clone(), 2, 3, 0.125, stream, kv=paged)
    assert hip.mi_hip_attn_fwd(ctypes.byref(args)) == 5
    assert hip.mi_hip_attn_fwd_reference_order(ctypes.byref(args)) == 5
    assert hip.mi_hip_attn_decode_batch(ctypes.byref(args), 1, stream) == 5
    assert hip.mi_hip_attn_decode_batch_noalloc(ctypes.byref(args), 1, stream) == 5
    assert hip.mi_hip_attn_tree(ctypes.byref(args), None, 1, stream) == 5
    assert hip.mi_hip_rope_append(ctypes.byref(mh.rope_args(paged, 0, 0, d, 1e4, stream, x, x))) == 5
    assert hip.mi_hip_norm_rope_append(ctypes.byref(mh.norm_rope_args(paged, 0, 0, d, 1e4, stream, x, x))) == 5
    assert hip.mi_hip_kv_keep(paged, 0, (ctypes.c_int32 * 1)(1), 1, stream) == 5
    node = mh.make_tensor(x.data_ptr(), [d, 2, 48], [4, 256, 512])
    assert hip.mi_hip_kv_bind(paged, 0, 0, ctypes.byref(node)) == 5
    host = np.zeros((t, 2, d), np.float32)
    nb = (ctypes.c_size_t * 3)(4, 256, 512)
    assert hip.mi_hip_kv_write(paged, 0, 0, 0, t, host.ctypes.data, nb, 0, stream) == 5
    hip.check(hip.mi_hip_kv_destroy(paged))
    hip.check(hip.mi_hip_kv_destroy(plain))
