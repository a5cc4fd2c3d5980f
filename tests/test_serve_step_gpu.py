"""The serving operators together: a step with a tree of drafted tokens, checked against the same
tokens fed one at a time.

Feeding the accepted path token by token writes the same cache rows (bit for bit, the rows do not
depend on what they are written with) and gives the same attention up to the rounding of sums
(serve_ref.attention_tolerance)."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref
from test_kv8_gpu import dev, read

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.mark.parametrize("kind", [mh.MI_TYPE_F32, mh.MI_TYPE_F16, mh.MI_HIP_TYPE_Q8])
@pytest.mark.parametrize("d,hkv,rep", [(64, 2, 7), (128, 4, 2)])
def test_tree_step_against_one_token_at_a_time(hip, stream, kind, d, hkv, rep):
    import torch
    rng = np.random.default_rng([d, kind])
    h, layers, n_past, t, vocab = hkv * rep, 2, 150, 24, 5000
    bits, depth = ref.random_tree(rng, t, width=4)
    scale = float(np.float32(d ** -0.5))
    wq, wk = (dev((1 + 0.2 * rng.standard_normal(d)).astype(np.float32)) for _ in range(2))
    freq = (1e6 ** (-np.arange(0, d, 2, dtype=np.float64) / d)).astype(np.float32)
    prompt = [[dev(rng.standard_normal((n_past, n, d)).astype(np.float32)) for n in (hkv, hkv)] for _ in range(layers)]
    draft = [[rng.standard_normal((t, n, d)).astype(np.float32) for n in (h, hkv, hkv)] for _ in range(layers)]
    head = dev(rng.standard_normal((vocab, h * d)).astype(np.float32) * 0.05)
    masks = mh.tree_masks([dev(bits.view(np.int64))])
    keep_bits = dev(bits.view(np.int64))
    masks[0].bits = keep_bits.data_ptr()

    def make():
        kv = hip.kv_create(layers, n_past + t + 4, hkv, d, h, kind)
        for layer, (k, v) in enumerate(prompt):
            a = mh.norm_rope_args(kv, layer, 0, d, 1e6, stream, k, v, freq=freq, k_norm=wk, eps=EPS)
            hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
        return kv

    def step(kv, past, rows, pos, m):
        """Appends the draft's rows at `past` and attends, layer by layer; the outputs."""
        outs = []
        dpos = dev(pos.astype(np.int32))
        for layer in range(layers):
            q, k, v = (dev(x[rows]) for x in draft[layer])
            qr, out = torch.empty_like(q), torch.empty_like(q)
            a = mh.norm_rope_args(kv, layer, past, d, 1e6, stream, k, v, q=q, q_out=qr, pos=dpos, freq=freq, q_norm=wq,
                                  k_norm=wk, eps=EPS)
            hip.check(hip.mi_hip_norm_rope_append(ctypes.byref(a)))
            items = (mh.AttnArgs * 1)(mh.attn_args(qr, out, rep, past, scale, stream, kv=kv, layer=layer))
            hip.check(hip.mi_hip_attn_tree(items, m, 1, stream))
            torch.cuda.synchronize()
            outs.append((qr.cpu().numpy(), out))
        return outs

    kv = make()
    tree = step(kv, n_past, np.arange(t), n_past + depth, masks)
    # each node's greedy id, with a penalty on its own path's ids (here the nodes' numbers)
    logits = tree[-1][1].view(t, -1) @ head.t()
    paths = [[i for i in range(t) if int(bits[j, 0]) >> i & 1] for j in range(t)]
    off = np.concatenate([[0], np.cumsum([len(p) for p in paths])]).astype(np.int32)
    hist = dev(np.concatenate(paths).astype(np.int32))
    pen, ids = dev(np.tile(np.array([[1.3, 0.1, 0.1]], np.float32), (t, 1))), torch.empty(t, device="cuda", dtype=torch.int32)
    adjusted, doff = torch.empty_like(logits), dev(off)
    a = mh.logits_args(logits, adjusted, stream, penalties=pen, hist=hist, hist_off=doff, ids=ids)
    hip.check(hip.mi_hip_logits_adjust(ctypes.byref(a)))
    torch.cuda.synchronize()
    lg, ad, got_ids = logits.cpu().numpy(), adjusted.cpu().numpy(), ids.cpu().numpy()
    for j in range(t):
        want = ref.logits(lg[j], [1.3, 0.1, 0.1], paths[j], [], None)
        assert np.abs(ad[j] - want).max() <= 8 * 2.0 ** -24 * (np.abs(lg[j]).max() * 1.3 + 1.0)
        assert got_ids[j] == ad[j].argmax()

    # the deepest node's path is accepted
    path = np.array(paths[int(depth.argmax())])
    assert len(path) >= 4 and not np.array_equal(path, np.arange(len(path)))
    hip.kv_keep(kv, n_past, path, stream)

    # the same tokens one at a time
    one = make()
    n = n_past + len(path)
    for i, node in enumerate(path):
        res = step(one, n_past + i, np.array([node]), np.array([n_past + i]), None)
        for layer in range(layers):
            q, out = res[layer]
            assert np.array_equal(q[0], tree[layer][0][node])
            k, v = (read(hip, one, layer, w, 0, n_past + i + 1, hkv, d, stream) for w in (0, 1))
            seen = np.ones((1, n_past + i + 1), bool)
            tol = ref.attention_tolerance(q, k, v, seen, scale)
            want = ref.attention(q, k, v, seen, scale)[0]
            assert np.abs(out.cpu().numpy()[0] - want).max() <= tol
            assert np.abs(tree[layer][1].cpu().numpy()[node] - want).max() <= tol
    for layer in range(layers):
        for w in (0, 1):
            assert np.array_equal(read(hip, kv, layer, w, 0, n, hkv, d, stream), read(hip, one, layer, w, 0, n, hkv, d, stream))
    # and the next tree goes on from there
    more = step(kv, n, np.arange(4), n + depth[:4], None)
    again = step(one, n, np.arange(4), n + depth[:4], None)
    for (q0, o0), (q1, o1) in zip(more, again):
        assert np.array_equal(q0, q1) and torch.equal(o0, o1)
    for x in (kv, one):
        hip.check(hip.mi_hip_kv_destroy(x))
