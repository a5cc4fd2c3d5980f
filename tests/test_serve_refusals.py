"""More refusals of the serving entry points that need no GPU (see test_serve_abi.py)."""
import pytest

import mi_hip_attn as mh

P = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return mh.lib()


@pytest.mark.parametrize("stride", [1 << 26, (1 << 26) + 16, 1 << 31, 1 << 32, 1 << 58, 1 << 59, 1 << 60, 3 << 61, 1 << 63])
@pytest.mark.parametrize("name", ["k_nb", "v_nb"])
def test_tree_refuses_rows_too_far_apart(lib, name, stride):
    # among them strides whose 32-fold passes 2^64
    items = (mh.AttnArgs * 1)()
    a = items[0]
    a.k = a.v = a.q = a.out = P
    a.kv_type, a.head_dim, a.n_head_kv, a.n_head, a.n_rep = mh.MI_TYPE_F32, 64, 2, 14, 7
    a.k_nb[:] = a.v_nb[:] = (4, 256, 512)
    a.q_nb[:] = a.out_nb[:] = (4, 256, 256 * 14)
    a.n_past, a.n_tokens, a.scale, a.ws = 5, 3, 0.125, P  # (the workspace is never read)
    getattr(a, name)[2] = stride
    assert lib.mi_hip_attn_tree(items, None, 1, None) == 5 and "stride" in lib.last_error()


def test_builders_refuse_floats_for_whole_numbers_and_tensors_of_two_devices(lib):
    import torch
    z, i32 = torch.zeros, torch.int32
    k, q = z(3, 2, 64), z(3, 4, 64)
    x, off = z(4, 100), z(5, dtype=i32)
    there = torch.device("meta")
    with pytest.raises(ValueError):  # float positions
        mh.norm_rope_args(None, 0, 0, 64, 1e4, None, k, k, pos=z(3))
    with pytest.raises(ValueError):  # float words
        mh.tree_masks([z(5, 1, dtype=torch.float64)])
    lists = dict(penalties=z(4, 3), hist=z(7, dtype=i32), hist_off=off, bias_id=z(2, dtype=i32), bias=z(2), bias_off=off,
                 mask=z(4, 4, dtype=i32), ids=z(4, dtype=i32))
    mh.logits_args(x, x, None, **lists)
    for name in ("hist", "hist_off", "bias_id", "bias_off", "mask", "ids"):
        with pytest.raises(ValueError):
            mh.logits_args(x, x, None, **dict(lists, **{name: lists[name].float()}))
    for name in ("penalties", "bias"):
        with pytest.raises(ValueError):
            mh.logits_args(x, x, None, **dict(lists, **{name: lists[name].to(i32)}))
    for name in lists:  # addresses of another device's memory
        with pytest.raises(ValueError):
            mh.logits_args(x, x, None, **dict(lists, **{name: lists[name].to(there)}))
    for kw in (dict(q=q.to(there)), dict(q=q, q_out=q.to(there)), dict(pos=z(3, dtype=i32, device=there)),
               dict(q_norm=z(64, device=there)), dict(k_norm=z(64, device=there))):
        with pytest.raises(ValueError):
            mh.norm_rope_args(None, 0, 0, 64, 1e4, None, k, k, **kw)
    with pytest.raises(ValueError):
        mh.norm_rope_args(None, 0, 0, 64, 1e4, None, k, k.to(there))


def test_rows_of_the_cache_have_its_shape_and_lie_on_a_gpu(lib):
    import torch
    kv = mh.KvHandle(1 << 20, 2, 64)  # (an address that is never read)
    good = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="device"):
        lib.kv_write(kv, 0, 0, 0, good, None)
    with pytest.raises(ValueError, match="device"):
        lib.kv_read(kv, 0, 0, 0, good, None)
    for shape in ((3, 1, 64), (3, 2, 32), (3, 3, 64), (3, 128), (1, 3, 2, 64)):
        with pytest.raises(ValueError, match="shape"):
            lib.kv_write(kv, 0, 0, 0, torch.zeros(shape), None)
        with pytest.raises(ValueError, match="shape"):
            lib.kv_read(kv, 0, 0, 0, torch.zeros(shape), None)
    for shape in ((3, 1, 64), (3, 4, 64), (3, 2, 128)):
        with pytest.raises(ValueError, match="shape"):
            mh.norm_rope_args(kv, 0, 0, 32, 1e4, None, torch.zeros(shape), torch.zeros(shape))
    mh.norm_rope_args(kv, 0, 0, 32, 1e4, None, good, good)
