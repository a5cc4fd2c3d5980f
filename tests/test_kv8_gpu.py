"""The 8-bit cache against its definition in 64 bits: the form is a function of the written values
(scale: the smallest f16 number with 127 d >= max |x|; value: the nearest whole number of x / d, ties
to even), so every comparison is exact."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import serve_ref as ref

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class _Mem:
    def __init__(self, ptr, shape, kind):
        self.__cuda_array_interface__ = dict(data=(ptr, False), shape=shape, typestr=kind, version=3)


def tensor_at(ptr, shape, kind):
    import torch
    return torch.as_tensor(_Mem(ptr, shape, kind), device="cuda")


def read(hip, kv, layer, which, pos0, n, hkv, d, stream, half=False):
    import torch
    out = torch.full((n, hkv, d), float("nan"), device="cuda", dtype=torch.float16 if half else torch.float32)
    hip.kv_read(kv, layer, which, pos0, out, stream)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def ties(d_, shape):
    """Values halfway between two steps of an f16 scale, the largest 127 steps."""
    k = np.arange(np.prod(shape)).reshape(shape) % 126
    x = (k + 0.5) * d_
    x[..., 0] = 127 * d_
    return x.astype(np.float32)


@pytest.mark.parametrize("d,hkv,n,pos0", [(64, 2, 1, 0), (128, 4, 7, 3), (64, 3, 130, 11), (128, 1, 33, 0)])
@pytest.mark.parametrize("kind", ["normal", "outliers", "ties", "tiny", "zeros", "large"])
def test_write_and_read_back(hip, stream, d, hkv, n, pos0, kind):
    rng = np.random.default_rng([d, hkv, n])
    x = rng.standard_normal((n, hkv, d)).astype(np.float32)
    if kind == "outliers":
        x[..., ::17] *= 300
    elif kind == "ties":
        x = ties(np.float32(0.0078125 * 3), x.shape)
    elif kind == "tiny":
        x *= np.float32(10.0) ** rng.integers(-12, -2, (n, hkv, 1)).astype(np.float32)
    elif kind == "zeros":
        x[::2] = 0
        x[1::2, :, 1:] = 0
    elif kind == "large":
        x *= 2e6 / np.abs(x).max()
    kv = hip.kv_create(2, pos0 + n + 2, hkv, d, hkv, mh.MI_HIP_TYPE_Q8)
    for which in (0, 1):
        hip.kv_write(kv, 1, which, pos0, dev(x), stream)
        got = read(hip, kv, 1, which, 0, pos0 + n + 2, hkv, d, stream)
        want = np.zeros(got.shape, np.float32)  # rows around stay the zeros of a new cache
        want[pos0:pos0 + n] = ref.q8(x, which)
        assert np.array_equal(got, want)
        assert np.abs(got[pos0:pos0 + n] - x).max() <= np.nanmax(ref.quantize(x, 32 if which == 0 else d)[1]) / 2
        half = read(hip, kv, 1, which, pos0, n, hkv, d, stream, half=True)
        assert np.array_equal(half, want[pos0:pos0 + n].astype(np.float16))
        assert not read(hip, kv, 0, which, 0, pos0 + n + 2, hkv, d, stream).any()  # the other layer
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_views_of_values_and_scales(hip, stream):
    import torch
    rng = np.random.default_rng(1)
    d, hkv, n = 128, 2, 5
    kv = hip.kv_create(3, n, hkv, d, hkv, mh.MI_HIP_TYPE_Q8)
    for layer in range(3):
        for which in (0, 1):
            x = rng.standard_normal((n, hkv, d)).astype(np.float32)
            hip.kv_write(kv, layer, which, 0, dev(x), stream)
            torch.cuda.synchronize()
            q, sc = ref.quantize(x, 32 if which == 0 else d)
            ptr, ne, nb = hip.kv_view(kv, layer, which)
            assert ne == [d, hkv, n, 1] and nb == [1, d, d * hkv, d * hkv * n]
            assert np.array_equal(tensor_at(ptr, (n, hkv, d), "|i1").cpu().numpy(), q.reshape(n, hkv, d))
            ptr, ne, nb = hip.kv_scales(kv, layer, which)
            g = d // 32 if which == 0 else 1
            assert ne == [g, hkv, n, 1] and nb == [2, 2 * g, 2 * g * hkv, 2 * g * hkv * n]
            assert np.array_equal(tensor_at(ptr, (n, hkv, g), "<f2").cpu().numpy(), sc)
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_groups_without_a_scale_read_as_nan(hip, stream):
    d, hkv, n = 64, 1, 5
    x = np.ones((n, hkv, d), np.float32)
    x[0, 0, 40] = np.inf
    x[1, 0, 3] = np.nan
    x[2, 0, 33] = -8319009.0   # 127 times the largest f16 number is 8319008
    x[3, 0, 33] = -8319008.0
    kv = hip.kv_create(1, n, hkv, d, hkv, mh.MI_HIP_TYPE_Q8)
    for which in (0, 1):
        hip.kv_write(kv, 0, which, 0, dev(x), stream)
        got = read(hip, kv, 0, which, 0, n, hkv, d, stream)
        bad = np.zeros((n, d), bool)
        if which == 0:
            bad[0, 32:], bad[1, :32], bad[2, 32:] = True, True, True
        else:
            bad[:3] = True
        assert np.array_equal(np.isnan(got[:, 0]), bad)
        assert np.array_equal(got[3:], ref.q8(x[3:], which))
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_strided_and_host_sources(hip, stream):
    import torch
    rng = np.random.default_rng(2)
    d, hkv, n = 64, 2, 9
    x = rng.standard_normal((n, hkv, d)).astype(np.float32)
    kv = hip.kv_create(1, n, hkv, d, hkv, mh.MI_HIP_TYPE_Q8)
    wide = torch.full((n, hkv + 1, d + 1), float("nan"), device="cuda")
    wide[:, :hkv, :d] = dev(x)
    hip.kv_write(kv, 0, 0, 0, wide[:, :hkv, :d], stream)
    assert np.array_equal(read(hip, kv, 0, 0, 0, n, hkv, d, stream), ref.q8(x, 0))
    turned = dev(x.transpose(2, 0, 1)).permute(1, 2, 0)  # dims far apart
    hip.kv_write(kv, 0, 1, 0, turned, stream)
    assert np.array_equal(read(hip, kv, 0, 1, 0, n, hkv, d, stream), ref.q8(x, 1))
    y = np.ascontiguousarray(x[::-1])
    hip.check(hip.mi_hip_kv_write(kv, 0, 0, 0, n, y.ctypes.data, (ctypes.c_size_t * 3)(4, 4 * d, 4 * d * hkv), 0, stream))
    assert np.array_equal(read(hip, kv, 0, 0, 0, n, hkv, d, stream), ref.q8(y, 0))
    # a strided destination keeps what lies between
    out = torch.full((n, hkv, 2 * d), -3.0, device="cuda")
    hip.kv_read(kv, 0, 0, 0, out[:, :, ::2], stream)
    torch.cuda.synchronize()
    assert np.array_equal(out[:, :, ::2].cpu().numpy(), ref.q8(y, 0)) and torch.all(out[:, :, 1::2] == -3.0)
    hip.check(hip.mi_hip_kv_destroy(kv))


@pytest.mark.parametrize("kind", [mh.MI_TYPE_F32, mh.MI_TYPE_F16])
def test_read_of_the_other_caches(hip, stream, kind):
    rng = np.random.default_rng(3)
    d, hkv, n = 128, 3, 6
    x = rng.standard_normal((n, hkv, d)).astype(np.float32)
    kv = hip.kv_create(1, n + 1, hkv, d, hkv, kind)
    hip.kv_write(kv, 0, 1, 1, dev(x), stream)
    held = x if kind == mh.MI_TYPE_F32 else x.astype(np.float16).astype(np.float32)
    assert np.array_equal(read(hip, kv, 0, 1, 1, n, hkv, d, stream), held)
    assert np.array_equal(read(hip, kv, 0, 1, 1, n, hkv, d, stream, half=True), x.astype(np.float16))
    hip.check(hip.mi_hip_kv_destroy(kv))


@pytest.mark.parametrize("kind", [mh.MI_TYPE_F32, mh.MI_TYPE_F16, mh.MI_HIP_TYPE_Q8])
@pytest.mark.parametrize("idx", [[0], [1], [2, 3, 4], [0, 1, 5, 9, 30], list(range(40)), [], list(range(1, 41)), [40]])
def test_keep(hip, stream, kind, idx):
    rng = np.random.default_rng(4)
    d, hkv, n_past, n, layers = 64, 3, 7, 41, 2
    kv = hip.kv_create(layers, n_past + n, hkv, d, hkv, kind)
    before = {}
    for layer in range(layers):
        for which in (0, 1):
            x = rng.standard_normal((n_past + n, hkv, d)).astype(np.float32)
            hip.kv_write(kv, layer, which, 0, dev(x), stream)
            before[layer, which] = read(hip, kv, layer, which, 0, n_past + n, hkv, d, stream)
    hip.kv_keep(kv, n_past, idx, stream)
    for (layer, which), was in before.items():
        want = was.copy()
        for i, j in enumerate(idx):
            want[n_past + i] = was[n_past + j]
        assert np.array_equal(read(hip, kv, layer, which, 0, n_past + n, hkv, d, stream), want)
    hip.check(hip.mi_hip_kv_destroy(kv))


def test_refusals(hip, stream):
    import torch
    kv = hip.kv_create(1, 8, 2, 64, 4, mh.MI_TYPE_F32)
    p = ctypes.c_void_p()
    assert hip.mi_hip_kv_scales(kv, 0, 0, ctypes.byref(p), None, None) == 5
    out = torch.zeros((8, 2, 64), device="cuda")
    nb = (ctypes.c_size_t * 3)(4, 256, 512)
    for layer, which, pos0, n, kind, code in [(1, 0, 0, 1, 0, 1), (0, 2, 0, 1, 0, 1), (0, 0, -1, 1, 0, 1),
                                              (0, 0, 0, 9, 0, 1), (0, 0, 8, 1, 0, 1), (0, 0, 0, 1, 2, 5),
                                              (0, 0, 2 ** 31 - 1, 2 ** 31 - 1, 0, 1), (0, 0, 0, -1, 0, 1)]:
        assert hip.mi_hip_kv_read(kv, layer, which, pos0, n, out.data_ptr(), kind, nb, stream) == code
    assert hip.mi_hip_kv_read(kv, 0, 0, 0, 1, out.data_ptr() + 2, 0, nb, stream) == 1
    assert hip.mi_hip_kv_read(kv, 0, 0, 0, 0, out.data_ptr(), 0, nb, stream) == 0
    for n_past, idx, code in [(0, [1, 1], 1), (0, [2, 1], 1), (0, [-1], 1), (0, [8], 1), (7, [1], 1), (9, [], 1),
                              (-1, [0], 1), (0, list(range(257)), 5)]:
        assert hip.mi_hip_kv_keep(kv, n_past, (ctypes.c_int32 * 300)(*idx), len(idx), stream) == code, (n_past, idx)
    hip.check(hip.mi_hip_kv_destroy(kv))
