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
