"""Penalties, biases, masks and greedy ids (mi_hip_logits_adjust) against 64 bits.

At most five roundings of float stand between the value and its 64-bit form (quotient or product,
count * frequency, + presence, -, + bias), and the biases' own sum: with e = 2^-24 the error is at most
8 e times the sum of the magnitudes that were added."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref
from test_kv8_gpu import dev

pytestmark = pytest.mark.gpu


def csr(lists, dtype):
    off = np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32)
    flat = np.concatenate([np.asarray(x, dtype) for x in lists]) if off[-1] else np.zeros(0, dtype)
    return flat.astype(dtype), off


def call(hip, stream, x, pen=None, hist=None, bias=None, mask=None, ids=True, out=None, nb=None, ws=None):
    """x: device rows; hist: lists; bias: lists of (id, value); mask: uint32 (rows, words)."""
    import torch
    n = x.shape[0]
    res = torch.full_like(x, float("nan")) if out is None else out
    dids = torch.full((n,), -9, device="cuda", dtype=torch.int32) if ids else None
    keep = {}
    if pen is not None:
        keep["penalties"] = dev(np.asarray(pen, np.float32))
    if hist is not None:
        f, o = csr(hist, np.int32)
        keep.update(hist=dev(f), hist_off=dev(o))
    if bias is not None:
        f, o = csr([[b[0] for b in r] for r in bias], np.int32)
        g, _ = csr([[b[1] for b in r] for r in bias], np.float32)
        keep.update(bias_id=dev(f), bias=dev(g), bias_off=dev(o))
    if mask is not None:
        keep["mask"] = dev(mask.view(np.int32))
    a = mh.logits_args(x, res, stream, ids=dids, ws=ws, **keep)
    hip.check(hip.mi_hip_logits_adjust(ctypes.byref(a)))
    torch.cuda.synchronize()
    return res.cpu().numpy(), dids.cpu().numpy() if ids else None


def check(x, got, ids, pen, hist, bias, allowed):
    for r in range(x.shape[0]):
        p = pen[r] if pen is not None else None
        h = hist[r] if hist is not None and p is not None else []
        b = bias[r] if bias is not None else []
        al = allowed[r] if allowed is not None else None
        want = ref.logits(x[r], p, h, b, al)
        size = np.abs(x[r].astype(np.float64))
        for t in h:
            if 0 <= t < len(size):
                size[t] = max(size[t], abs(float(x[r, t])) * max(float(p[0]), 1 / float(p[0]))) + abs(float(p[1])) + abs(float(p[2]))
        for t, v in b:
            if 0 <= t < len(size):
                size[t] += abs(float(v))
        fin = np.isfinite(want)
        assert np.array_equal(got[r][~fin], want[~fin].astype(np.float32), equal_nan=True)
        assert np.all(np.abs(got[r][fin] - want[fin]) <= 8 * 2.0 ** -24 * size[fin] + 2.0 ** -149)
        if ids is not None:  # the rule, on the row as it came out
            ok = got[r] > -np.inf
            assert ids[r] == (int(np.argmax(np.where(ok, got[r], -np.inf))) if ok.any() else -1)


@pytest.mark.parametrize("vocab,rows", [(1, 1), (31, 2), (33, 3), (1000, 5), (4096, 2), (4097, 3), (8195, 1), (32000, 70),
                                        (151936, 2)])
@pytest.mark.parametrize("what", ["plain", "hist", "bias", "mask", "all"])
def test_against_64_bits(hip, stream, vocab, rows, what):
    rng = np.random.default_rng([vocab, rows])
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    pen = hist = bias = mask = allowed = None
    if what in ("hist", "all"):
        pen = np.stack([1 + rng.random(rows), rng.random(rows) - 0.3, rng.random(rows)], 1).astype(np.float32)
        # lists of their own lengths, empty ones, repeated ids, ids that are none
        hist = [list(rng.integers(0, vocab, int(rng.integers(0, 300)))) + [-1, vocab, 2 ** 31 - 1, -2 ** 31] * (r % 2)
                for r in range(rows)]
        hist[0] = [vocab // 2] * 70 + [0, vocab - 1]
    if what in ("bias", "all"):
        bias = [[(int(t), float(np.float32(rng.standard_normal() * 4))) for t in rng.integers(0, vocab, r % 7)]
                + [(-5, 1.0), (vocab, 1.0)] for r in range(rows)]
    if what in ("mask", "all"):
        words = (vocab + 31) // 32
        mask = rng.integers(0, 2 ** 32, (rows, words), dtype=np.uint32)
        mask[0, ::2] = 0
        if rows > 1:
            mask[1] = 0  # nothing is allowed
        allowed = np.unpackbits(mask.view(np.uint8), axis=1, bitorder="little")[:, :vocab].astype(bool)
    got, ids = call(hip, stream, dev(x), pen, hist, bias, mask)
    check(x, got, ids, pen, hist, bias, allowed)
    if what == "plain":
        assert np.array_equal(got, x)


def test_the_same_token_listed_many_times(hip, stream):
    # a bias list's order decides the sum: the same bits every time
    x = np.zeros((1, 5000), np.float32)
    bias = [[(17, 1e8), (17, 1.0), (4500, 0.5), (17, -1e8), (17, 3.0)] * 40]
    want = np.float32(0)
    for t, v in bias[0]:
        if t == 17:
            want = np.float32(want + np.float32(v))
    for _ in range(5):
        got, _ = call(hip, stream, dev(x), bias=bias)
        assert got[0, 17] == want and got[0, 4500] == np.float32(20.0)
    pen = [[1.5, 0.25, 0.125]]
    got, _ = call(hip, stream, dev(x + 3), pen=pen, hist=[[2999] * 100000])
    assert got[0, 2999] == np.float32(3 / 1.5) - np.float32(100000 * 0.25 + 0.125)


def test_ids_of_ties_infinities_and_nan(hip, stream):
    n = 9000
    x = np.full((8, n), -1.0, np.float32)
    x[0, [5000, 8000, 4999]] = 2.0            # ties across chunks: the lowest
    x[1, 100], x[1, 50] = np.inf, np.nan      # NaN is never chosen
    x[2] = -np.inf
    x[3] = np.nan
    x[4, 1:] = -np.inf
    x[5] = -0.0
    x[5, 7] = 0.0                             # zeros are equal
    x[6] = np.finfo(np.float32).min
    x[7, n - 1] = 1e-45
    _, ids = call(hip, stream, dev(x))
    assert list(ids) == [4999, 100, -1, -1, 0, 0, 0, n - 1]


def test_in_place_strided_one_mask_for_all_and_no_ids(hip, stream):
    import torch
    rng = np.random.default_rng(5)
    rows, vocab = 6, 1003
    buf = torch.full((rows, vocab + 5), -7.0, device="cuda")
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    view = buf[:, 1:vocab + 1]
    view.copy_(dev(x))
    mask = rng.integers(0, 2 ** 32, (1, (vocab + 31) // 32), dtype=np.uint32)
    allowed = np.repeat(np.unpackbits(mask.view(np.uint8), axis=1, bitorder="little")[:, :vocab].astype(bool), rows, 0)
    pen = np.tile(np.array([[1.3, 0.1, 0.2]], np.float32), (rows, 1))
    hist = [list(rng.integers(0, vocab, 50)) for _ in range(rows)]
    got, ids = call(hip, stream, view, pen, hist, mask=mask, out=view)
    check(x, got, ids, pen, hist, None, allowed)
    assert torch.all(buf[:, 0] == -7.0) and torch.all(buf[:, vocab + 1:] == -7.0)
    got2, none = call(hip, stream, dev(x), pen, hist, mask=mask, ids=False)
    assert none is None and np.array_equal(got2, got)


def test_more_rows_than_the_scratch_holds_at_once(hip, stream):
    # a launch takes as many rows as their chunks' maxima have room for
    rng = np.random.default_rng(6)
    rows, vocab = 70000, 33
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    hist = [[r % vocab] * (r % 3) for r in range(rows)]
    pen = np.tile(np.array([[2.0, 0.5, 0.25]], np.float32), (rows, 1))
    got, ids = call(hip, stream, dev(x), pen, hist)
    want = x.copy()
    for r in range(rows):
        c, t = r % 3, r % vocab
        if c:
            y = x[r, t] / np.float32(2) if x[r, t] > 0 else x[r, t] * np.float32(2)
            want[r, t] = y - (np.float32(c) * np.float32(0.5) + np.float32(0.25))
    assert np.array_equal(got, want) and np.array_equal(ids, want.argmax(1))


def test_captured_and_replayed(hip, stream):
    import torch
    rng = np.random.default_rng(7)
    rows, vocab = 4, 20000
    x = dev(rng.standard_normal((rows, vocab)).astype(np.float32))
    pen = dev(np.tile(np.array([[1.3, 0.1, 0.2]], np.float32), (rows, 1)))
    f, o = csr([list(rng.integers(0, vocab, 99)) for _ in range(rows)], np.int32)
    hist, off = dev(f), dev(o)
    out, ids = torch.empty_like(x), torch.empty(rows, device="cuda", dtype=torch.int32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        a = mh.logits_args(x, out, torch.cuda.current_stream().cuda_stream, penalties=pen, hist=hist, hist_off=off, ids=ids)
        hip.check(hip.mi_hip_logits_adjust(ctypes.byref(a)))
    for seed in range(4):
        x.copy_(dev(np.random.default_rng(seed).standard_normal((rows, vocab)).astype(np.float32)))
        out.fill_(0)
        ids.fill_(-5)
        g.replay()
        torch.cuda.synchronize()
        got, gid = out.cpu().numpy(), ids.cpu().numpy()
        want, wid = torch.empty_like(x), torch.empty_like(ids)
        b = mh.logits_args(x, want, stream, penalties=pen, hist=hist, hist_off=off, ids=wid)
        hip.check(hip.mi_hip_logits_adjust(ctypes.byref(b)))
        torch.cuda.synchronize()
        assert np.array_equal(got, want.cpu().numpy()) and np.array_equal(gid, wid.cpu().numpy())
