"""Plain 64-bit forms of the serving operators, for their tests."""
import math

import numpy as np


def visible(n_past, n_tok, bits=None):
    """(n_tok, n_past + n_tok) truth values; bits: uint64 words (n_tok, words) or None for a chain."""
    v = np.ones((n_tok, n_past + n_tok), dtype=bool)
    for j in range(n_tok):
        for i in range(n_tok):
            v[j, n_past + i] = i <= j if bits is None else bool(int(bits[j, i // 64]) >> (i % 64) & 1)
    return v


def attention(q, k, v, seen, scale):
    """softmax(scale q.k) v over the seen keys, in 64 bits; zeros for a row that sees none.
    q (t, h, d), k and v (n_kv, hkv, d), seen (t, n_kv)."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    h = q.shape[1]
    rep = h // k.shape[1]
    out = np.zeros(q.shape)
    for i in range(h):
        s = np.where(seen, q[:, i] @ k[:, i // rep].T * scale, -np.inf)
        top = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
        total = p.sum(1, keepdims=True)
        out[:, i] = p @ v[:, i // rep] / np.where(total > 0, total, 1.0)
    return out


def attention_tolerance(q, k, v, seen, scale):
    """The most that a correct kernel's output may be off. With e = 2^-24: a score is a sum of d
    products of 24-bit operands (or of f16 pairs, 2^-22 off) accumulated in float, scaled and
    turned to base 2, so it is at most (d + 12) e S off, S = scale sum |q||k|; that moves an output
    by at most twice as much of the largest |v| it averages. The sums over keys, the exponentials and
    the joins add at most one rounding per 32-key tile and join and a dozen more."""
    q, k = np.abs(q.astype(np.float64)), np.abs(k.astype(np.float64))
    vm = np.abs(v[seen.any(0)].astype(np.float64)).max(initial=0.0)
    t, h, d = q.shape
    rep = h // k.shape[1]
    s = 0.0
    used = k[seen.any(0)]
    for i in range(h):
        if len(used):
            s = max(s, float((used[:, i // rep] @ q[:, i].T).max()) * abs(scale))
    e = 2.0 ** -24
    return vm * e * (2 * (d + 12) * s + k.shape[0] / 32 + 32 * 16)


def f16_scale(amax):
    """The smallest f16 number d with 127 d >= amax (float64 in and out; inf past the range)."""
    a = np.asarray(amax, np.float64) / 127.0
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.maximum(a, 2.0 ** -14)))
        step = np.exp2(e - 10)
        d = np.ceil(a / step) * step
        # 127 d >= amax must hold for the exact product, and not for the number below
        low = d - step
        d = np.where((low > 0) & (127.0 * low >= amax), low, d)
        return np.where(d > 65504.0, np.where(np.isnan(d), d, np.inf), d)


def quantize(x, group):
    """(whole numbers, scales) of the 8-bit form of the rows of x, NaN scales for groups without one."""
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, group)
    amax = np.abs(g).max(-1)
    d = f16_scale(amax)
    d = np.where(np.isfinite(d), d, np.nan)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(d[..., None] > 0, np.rint(g / np.where(d > 0, d, 1.0)[..., None]), 0.0)
    return q, d


def stands_for(q, d):
    return (q * d[..., None]).reshape(*q.shape[:-2], -1)


def q8(x, which):
    """What K (which 0) or V (1) rows read back as from an 8-bit cache."""
    return stands_for(*quantize(x, 32 if which == 0 else x.shape[-1]))


def norm_rope(x, w, eps, pos, freq):
    """Rows (t, h, d) normed per head (w or None), the first 2 len(freq) dims rotated by the float
    product pos * freq; 64 bits otherwise."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    half = len(freq)
    theta = (pos.astype(np.float32)[:, None] * freq.astype(np.float32)[None, :]).astype(np.float64)[:, None, :]
    a, b = y[..., :half].copy(), y[..., half:2 * half].copy()
    y = y.copy()
    y[..., :half] = a * np.cos(theta) - b * np.sin(theta)
    y[..., half:2 * half] = a * np.sin(theta) + b * np.cos(theta)
    return y


def logits(x, penalties, hist, bias, allowed):
    """One row in 64 bits: penalties (repeat, frequency, presence) or None, hist ids, bias [(id, value)],
    allowed truth values or None."""
    y = x.astype(np.float64).copy()
    n = len(y)
    for t in set(h for h in hist if 0 <= h < n):
        c = sum(1 for h in hist if h == t)
        rep, freq, pres = (float(p) for p in penalties)
        y[t] = (y[t] / rep if y[t] > 0 else y[t] * rep) - (c * freq + pres)
    for t, v in bias:
        if 0 <= t < n:
            y[t] += float(v)
    if allowed is not None:
        y[~allowed] = -math.inf
    return y


def random_tree(rng, n, width=8):
    """Parents' bits of a random tree: uint64 words (n, words), and depths."""
    words = (n + 63) // 64
    seen, depth = [], np.zeros(n, np.int32)
    bits = np.zeros((n, words), np.uint64)
    for i in range(n):
        p = int(rng.integers(max(-1, i - width), i)) if i else -1
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        depth[i] = depth[p] + 1 if p >= 0 else 0
        for w in range(words):
            bits[i, w] = seen[i] >> 64 * w & 0xFFFFFFFFFFFFFFFF
    return bits, depth
