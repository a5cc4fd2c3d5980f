"""Refusals of the entry points over a paged cache that need no GPU: they come before any device
work, so the addresses below are never touched."""
import ctypes

import pytest

import mi_hip_attn as mh

P = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return mh.lib()


def rc_of(lib, name, args, **kw):
    for n, v in kw.items():
        if n.endswith("_nb") and not isinstance(v, int):
            getattr(args, n)[:] = v
        else:
            setattr(args, n, v)
    return getattr(lib, name)(ctypes.byref(args))


def tables(**kw):
    a = mh.PageTablesArgs()
    a.n_seq, a.page_size, a.n_pages, a.max_pages, a.max_tokens, a.table_nb = 4, 16, 100, 10, 50, 40
    for n in ("n_cached", "n_new", "held", "held_out", "table", "ring", "ring_at", "ring_at_out", "n_kv", "q_off", "slots"):
        setattr(a, n, P)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(n_seq=-1), 1), (dict(max_tokens=-1), 1), (dict(n_pages=0), 1), (dict(max_pages=0), 1), (dict(page_size=0), 5),
    (dict(page_size=8), 5), (dict(page_size=24), 5), (dict(page_size=-16), 5), (dict(page_size=-2 ** 31), 5),
    (dict(n_pages=1 << 28), 5), (dict(max_pages=1 << 27, table_nb=1 << 29), 5), (dict(n_new=None), 1), (dict(slots=None), 1),
    (dict(held=P + 2), 1), (dict(pos=P + 1), 1), (dict(seq=P + 2), 1), (dict(n_refused=P + 3), 1), (dict(table_nb=36), 1),
    (dict(table_nb=42), 1), (dict(), 6)])
def test_page_tables(lib, kw, code):
    assert lib.mi_hip_page_tables(None) == 1
    got = rc_of(lib, "mi_hip_page_tables", tables(), **kw)
    assert got == code or (code == 6 and no_device_answer(got)), lib.last_error()


def no_device_answer(rc):
    """A call that passes its checks where no device is: refused as uninitialised."""
    import torch
    return torch.cuda.is_available() or rc == 6


def test_calls_without_a_cache(lib):
    for name, args in (("mi_hip_paged_append", mh.PagedAppendArgs()), ("mi_hip_attn_paged", mh.AttnPagedArgs())):
        assert getattr(lib, name)(None) == 1 and "NULL" in lib.last_error()
        assert getattr(lib, name)(ctypes.byref(args)) == 1 and "NULL" in lib.last_error()


@pytest.mark.parametrize("desc,page,code", [
    ((2, 64, 2, 64, 14, 0), 8, 5), ((2, 64, 2, 64, 14, 0), 48, 5), ((2, 64, 2, 64, 14, 0), 0, 5), ((2, 72, 2, 64, 14, 0), 16, 1),
    ((2, 64, 2, 64, 13, 0), 16, 1), ((2, 64, 2, 96, 14, 0), 16, 5), ((2, 64, 2, 64, 14, 2), 16, 5), ((0, 64, 2, 64, 14, 0), 16, 1)])
def test_kv_create_paged(lib, desc, page, code):
    h = ctypes.c_void_p()
    assert lib.mi_hip_kv_create_paged(ctypes.byref(mh.KvDesc(*desc)), page, ctypes.byref(h)) == code and not h.value
    assert lib.mi_hip_kv_create_paged(None, 16, ctypes.byref(h)) == 1


def verify(**kw):
    a = mh.VerifyArgs()
    a.n_vocab, a.n_rows, a.n_seq, a.max_path, a.nb, a.draft_nb, a.path_nb, a.tokens_nb = 100, 8, 2, 5, 400, 400, 20, 20
    for n in ("logits", "off", "token", "u", "n_path", "path", "tokens"):
        setattr(a, n, P)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(n_vocab=0), 1), (dict(n_rows=-1), 1), (dict(n_seq=-1), 1), (dict(max_path=0), 1), (dict(n_vocab=2 ** 31 - 1, nb=2 ** 34), 5),
    (dict(off=None), 1), (dict(u=None), 1), (dict(token=None), 1), (dict(tokens=None), 1), (dict(n_path=None), 1),
    (dict(draft=P, parent=P), 5), (dict(nb=396), 1), (dict(nb=402), 1), (dict(draft=P, draft_nb=396), 1),
    (dict(draft=P, draft_nb=401), 1), (dict(path_nb=16), 1), (dict(tokens_nb=22), 1), (dict(logits=P + 2), 1),
    (dict(parent=P + 1), 1), (dict(temperature=P + 2), 1), (dict(), 6), (dict(n_rows=1, nb=0), 6)])
def test_verify(lib, kw, code):
    assert lib.mi_hip_verify_draft(None) == 1
    got = rc_of(lib, "mi_hip_verify_draft", verify(), **kw)
    assert got == code or (code == 6 and no_device_answer(got)), lib.last_error()


def test_builders(lib):
    import torch
    z, i32 = torch.zeros, torch.int32
    n, t = 3, 10
    lens = dict(n_cached=z(n, dtype=i32), n_new=z(n, dtype=i32), held=z(n, dtype=i32), held_out=z(n, dtype=i32),
                table=z(n, 4, dtype=i32), ring=z(20, dtype=i32), ring_at=z(2, dtype=i32), ring_at_out=z(2, dtype=i32),
                n_kv=z(n, dtype=i32), q_off=z(n + 1, dtype=i32), slots=z(t, dtype=i32), pos=z(t, dtype=i32),
                seq=z(t, dtype=i32), n_refused=z(1, dtype=i32))
    a = mh.page_tables_args(16, stream=None, **lens)
    assert (a.n_seq, a.n_pages, a.max_pages, a.max_tokens, a.table_nb) == (3, 20, 4, 10, 16)
    for name in lens:
        for other in (lens[name].float(), z(7, dtype=i32), lens[name].to("meta")):
            if name == "slots" and other.shape == (7,):
                continue  # (their number is the call's: pos and seq then differ, tested by those)
            if name == "ring" and other.shape == (7,) or name == "n_refused" and other.shape == (7,):
                continue
            with pytest.raises(ValueError):
                mh.page_tables_args(16, stream=None, **dict(lens, **{name: other}))
    k, q, s = z(t, 2, 64), z(t, 4, 64), z(t, dtype=i32)
    pos = z(3, t, dtype=i32)
    mh.paged_append_args(None, 0, 64, 1e4, None, k, k, s, pos, q=q, axis=[0] * 32)
    for kw in (dict(slots=s.float()), dict(slots=s[:5]), dict(pos=z(5, t, dtype=i32)), dict(pos=pos.float()),
               dict(pos=pos[:, :4]), dict(axis=[0] * 31), dict(v=k.to("meta"))):
        with pytest.raises(ValueError):
            mh.paged_append_args(None, 0, 64, 1e4, None, **dict(dict(k=k, v=k, slots=s, pos=pos, q=q), **kw))
    good = dict(q=q, out=q.clone(), q_off=z(n + 1, dtype=i32), n_kv=z(n, dtype=i32), table=z(n, 4, dtype=i32))
    mh.paged_attn_args(None, 0, scale=1.0, stream=None, **good)
    for kw in (dict(q=q.half()), dict(out=q[:5]), dict(q_off=z(n, dtype=i32)), dict(n_kv=z(n)), dict(table=z(n + 1, 4, dtype=i32)),
               dict(table=z(n, 8, dtype=i32)[:, ::2]), dict(out=q.to("meta"))):
        with pytest.raises(ValueError):
            mh.paged_attn_args(None, 0, scale=1.0, stream=None, **dict(good, **kw))
    with pytest.raises(ValueError):
        mh.paged_attn_args(mh.KvHandle(P, 2, 128), 0, scale=1.0, stream=None, **good)
    good = dict(logits=z(8, 100), off=z(3, dtype=i32), token=z(8, dtype=i32), u=z(8), n_path=z(2, dtype=i32),
                path=z(2, 5, dtype=i32), tokens=z(2, 5, dtype=i32), parent=z(8, dtype=i32), temperature=z(2))
    mh.verify_args(stream=None, **good)
    for kw in (dict(logits=z(8, 100).half()), dict(draft=z(8, 99)), dict(off=z(2, dtype=i32)), dict(token=z(8)), dict(u=z(7)),
               dict(temperature=z(3)), dict(path=z(2, 4, dtype=i32)), dict(tokens=z(2, 5)), dict(parent=z(7, dtype=i32)),
               dict(u=z(8, device="meta"))):
        with pytest.raises(ValueError):
            mh.verify_args(stream=None, **dict(good, **kw))


@pytest.mark.parametrize("n,code", [(1 << 30, 1), ((1 << 30) + 1, 5), (2 ** 31 - 1, 5)])
def test_page_tables_of_too_many_sequences(lib, n, code):
    # (as many as may be go on to the next check, of the table's rows)
    assert rc_of(lib, "mi_hip_page_tables", tables(), n_seq=n, table_nb=36) == code, lib.last_error()


@pytest.mark.parametrize("n,code", [(1 << 30, 1), ((1 << 30) + 1, 5), (2 ** 31 - 1, 5)])
def test_verification_of_too_many_sequences(lib, n, code):
    # (as many as may be go on to the next check, of the pointers)
    assert rc_of(lib, "mi_hip_verify_draft", verify(), n_seq=n, off=None) == code, lib.last_error()
