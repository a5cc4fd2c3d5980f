"""The serving operators at the ends of their ranges: values that are not finite in the first keys of
many workgroups, rows of very small values, positions far apart, sources of any alignment, caches and
workspaces under an allocation limit. References in 64 bits."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref
from test_kv8_gpu import dev, read
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
