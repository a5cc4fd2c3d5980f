"""Refusals of the serving entry points that need no GPU: they come before any device work, so the
addresses below are never touched."""
import ctypes

import pytest

import mi_hip_attn as mh

P = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return mh.lib()


def test_tree(lib):
    assert lib.mi_hip_attn_tree(None, None, 1, None) == 1
    items = (mh.AttnArgs * 1)()
    a = items[0]
    assert lib.mi_hip_attn_tree(items, None, 0, None) == 1

    def reset():
        a.k = a.v = a.q = a.out = P
        a.kv_type, a.head_dim, a.n_head_kv, a.n_head, a.n_rep = mh.MI_TYPE_F32, 64, 2, 14, 7
        a.k_nb[:] = a.v_nb[:] = (4, 256, 512)
        a.q_nb[:] = a.out_nb[:] = (4, 256, 256 * 14)
        a.n_past, a.n_tokens, a.scale = 5, 3, 0.125
        a.ws = P  # (never read: refused or uninitialised before)
    for name, value, code in [("head_dim", 80, 5), ("n_rep", 6, 1), ("n_tokens", 0, 1), ("n_past", -1, 1),
                              ("scale", float("inf"), 1), ("q", None, 1), ("out", P + 4, 5), ("k", None, 1),
                              ("kv_type", mh.MI_HIP_TYPE_Q8, 5), ("k_nb", (4, 256, 128), 5),
                              ("v_nb", (4, 256, 1 << 28), 5), ("n_past", 2 ** 31 - 10, 5), ("n_tokens", 1 << 23, 5)]:
        reset()
        if name.endswith("_nb"):
            getattr(a, name)[:] = value
        else:
            setattr(a, name, value)
        assert lib.mi_hip_attn_tree(items, None, 1, None) == code, (name, lib.last_error())
    reset()
    for bits, nb, code in [(P + 4, 8, 5), (P, 12, 5), (P, 0, 1)]:
        m = (mh.TreeMask * 1)(mh.TreeMask(bits, nb))
        assert lib.mi_hip_attn_tree(items, m, 1, None) == code
    two = (mh.AttnArgs * 2)(a, a)
    two[1].scale = 0.25
    assert lib.mi_hip_attn_tree(two, None, 2, None) == 1 and "item 1" in lib.last_error()


def test_logits(lib):
    def rc(**kw):
        a = mh.LogitsArgs()
        a.logits, a.out, a.nb, a.out_nb, a.n_vocab, a.n_rows = P, 2 * P, 400, 400, 100, 2
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.mi_hip_logits_adjust(ctypes.byref(a))
    assert lib.mi_hip_logits_adjust(None) == 1
    for kw, code in [(dict(logits=None), 1), (dict(out=None), 1), (dict(n_vocab=0), 1), (dict(n_rows=-1), 1),
                     (dict(nb=396), 1), (dict(out_nb=402), 1), (dict(logits=P + 2), 1), (dict(hist=P), 1),
                     (dict(hist=P, hist_off=P), 1), (dict(bias_id=P), 1), (dict(bias_id=P, bias=P), 1),
                     (dict(mask=P, mask_nb=8), 1), (dict(mask=P + 2), 1), (dict(ids=P + 1), 1),
                     (dict(out=P, out_nb=800), 1), (dict(n_vocab=2 ** 31 - 1, nb=2 ** 34, out_nb=2 ** 34), 5)]:
        assert rc(**kw) == code, kw
    assert rc(n_rows=0) == 0


def test_cache_handles(lib):
    x, nb = ctypes.c_void_p(), (ctypes.c_size_t * 3)(4, 256, 512)
    assert lib.mi_hip_kv_scales(None, 0, 0, ctypes.byref(x), None, None) == 1
    assert lib.mi_hip_kv_read(None, 0, 0, 0, 1, P, 0, nb, None) == 1
    assert lib.mi_hip_kv_keep(None, 0, None, 0, None) == 1
    assert lib.mi_hip_norm_rope_append(None) == 1
    a = mh.NormRopeArgs()
    assert lib.mi_hip_norm_rope_append(ctypes.byref(a)) == 1 and "NULL" in lib.last_error()


def test_builders_refuse_what_does_not_fit(lib):
    import torch
    f = torch.zeros
    q, k, v = f(3, 4, 64), f(3, 2, 64), f(3, 2, 64)
    i32 = torch.int32
    mh.norm_rope_args(None, 0, 0, 64, 1e4, None, k, v, q=q, pos=f(3, dtype=i32), q_norm=f(64), k_norm=f(64), freq=[1.0] * 32)
    for kw in (dict(q=q.half()), dict(q=q[:2]), dict(q=q[..., :32]), dict(q=q, q_out=q[:, :2]), dict(q_norm=f(32)),
               dict(k_norm=f(128)[::2]), dict(pos=f(2, dtype=i32)), dict(pos=f(3, dtype=torch.int64)), dict(freq=[1.0] * 31)):
        with pytest.raises(ValueError):
            mh.norm_rope_args(None, 0, 0, 64, 1e4, None, k, v, **kw)
    with pytest.raises(ValueError):
        mh.norm_rope_args(None, 0, 0, 64, 1e4, None, k, v.half())
    mh.tree_masks([None, f(5, 1, dtype=torch.int64), f(5, 3, dtype=torch.int64)[:, :1]])
    for bad in (f(5, 2, dtype=i32), f(5, dtype=torch.int64), f(2, 5, dtype=torch.int64).t()):
        with pytest.raises(ValueError):
            mh.tree_masks([bad])
    x, words = f(4, 100), f(4, 4, dtype=i32)
    off = f(5, dtype=i32)
    mh.logits_args(x, x, None, penalties=f(4, 3), hist=f(7, dtype=i32), hist_off=off, bias_id=f(2, dtype=i32), bias=f(2),
                   bias_off=off, mask=words, ids=f(4, dtype=i32))
    for kw in (dict(out=f(4, 99)), dict(out=x.half()), dict(out=f(100, 4).t()), dict(penalties=f(3, 3)),
               dict(hist_off=off[:4]), dict(hist=f(7, dtype=torch.int64)), dict(bias=f(2)),
               dict(bias=f(2), bias_id=f(3, dtype=i32)), dict(mask=words[:3]), dict(mask=words[:, :3]),
               dict(mask=words.to(torch.int64)), dict(ids=f(3, dtype=i32))):
        with pytest.raises(ValueError):
            mh.logits_args(x, kw.pop("out", x), None, **kw)
    for call in (lambda t: lib.kv_write(None, 0, 0, 0, t, None), lambda t: lib.kv_read(None, 0, 0, 0, t, None)):
        for bad in (k.double(), k.bfloat16(), k.to(torch.int16)):
            with pytest.raises(ValueError):
                call(bad)
    with pytest.raises(ValueError):
        lib.kv_write(None, 0, 0, 0, k.half(), None)
