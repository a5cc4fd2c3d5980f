"""Block tables and slot maps (mi_hip_page_tables) against a sequence-by-sequence form: whole numbers,
every comparison is exact."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import paged_ref as ref
from test_kv8_gpu import dev

pytestmark = pytest.mark.gpu


def state(rng, n, page, cached, new, held, free, extra=3, spare_tokens=3, width=None):
    """A pool in which the held pages are with their sequences, `free` in the ring, some with others."""
    n_pages = int(held.sum()) + free + extra
    ids = rng.permutation(n_pages)
    need = -(-(np.maximum(cached, 0) + np.maximum(new, 0)) // page)
    width = int(max(need.max(initial=1), held.max(initial=1), 1)) + 1 if width is None else width
    table = np.full((n, width), -1, np.int64)
    table[np.arange(width)[None, :] < held[:, None]] = ids[:held.sum()]
    head = int(rng.integers(0, n_pages))
    ring = np.full(n_pages, -7, np.int64)
    ring[(head + np.arange(free)) % n_pages] = ids[held.sum():held.sum() + free]
    total = int(np.maximum(new, 0).sum()) + spare_tokens
    return dict(page=page, n_pages=n_pages, max_pages=width, max_tokens=total, cached=cached, new=new, held=held, table=table,
                ring=ring, ring_at=np.array([head, head + free]))


class Call:
    def __init__(self, s, stream, in_place=False, max_tokens=None, table_pad=0):
        import torch
        i32 = lambda x: dev(np.asarray(x, np.int32))
        n, t = len(s["cached"]), s["max_tokens"] if max_tokens is None else max_tokens
        full = lambda m: torch.full((m,), -99, dtype=torch.int32, device="cuda")
        wide = np.full((n, s["max_pages"] + table_pad), -5, np.int32)
        wide[:, :s["max_pages"]] = s["table"]
        self.wide, self.width = dev(wide), s["max_pages"]
        self.inputs = dict(cached=i32(s["cached"]), new=i32(s["new"]), held=i32(s["held"]), ring_at=i32(s["ring_at"]))
        self.out = dict(held=self.inputs["held"] if in_place else full(n), table=self.wide[:, :s["max_pages"]], ring=i32(s["ring"]),
                        ring_at=self.inputs["ring_at"] if in_place else full(2), n_kv=full(n), q_off=full(n + 1),
                        slots=full(t), pos=full(t), seq=full(t), refused=full(1))
        i, o = self.inputs, self.out
        self.args = mh.page_tables_args(s["page"], i["cached"], i["new"], i["held"], o["held"], o["table"], o["ring"],
                                        i["ring_at"], o["ring_at"], o["n_kv"], o["q_off"], o["slots"], stream, pos=o["pos"],
                                        seq=o["seq"], n_refused=o["refused"])

    def got(self):
        import torch
        torch.cuda.synchronize()
        return {k: v.cpu().numpy().astype(np.int64) for k, v in self.out.items()}


def same(got, want):
    for k, w in want.items():
        assert np.array_equal(got[k], w), k


def requests(rng, n, page, most, chunk):
    cached = rng.integers(0, most + 1, n)
    new = rng.integers(0, chunk + 1, n)
    held = np.maximum(0, -(-cached // page) + rng.integers(-1, 3, n))
    end = rng.random(n) < 0.15
    cached[end], new[end] = 0, 0
    return cached, new, held


@pytest.mark.parametrize("n,page,most,chunk", [
    (1, 16, 0, 1), (1, 256, 100, 1), (3, 16, 40, 0), (8, 16, 600, 1), (63, 32, 100, 40), (64, 64, 3000, 1), (65, 16, 50, 300),
    (1000, 16, 500, 3), (1024, 128, 900, 40), (1025, 16, 100, 7), (4500, 32, 300, 20), (3, 16, 10, 30000), (40, 1 << 20, 50, 9)])
@pytest.mark.parametrize("free", ["enough", "tight", "none"])
@pytest.mark.parametrize("in_place", [False, True])
def test_against_the_plain_form(hip, stream, n, page, most, chunk, free, in_place):
    rng = np.random.default_rng([n, page, most, chunk])
    cached, new, held = requests(rng, n, page, most, chunk)
    taken = int(np.maximum(-(-(cached + new) // page) - held, 0).sum())
    s = state(rng, n, page, cached, new, held, dict(enough=taken, tight=taken // 2, none=0)[free])
    c = Call(s, stream, in_place, table_pad=2)
    hip.check(hip.mi_hip_page_tables(ctypes.byref(c.args)))
    same(c.got(), ref.page_tables(**s))
    assert bool((c.wide[:, c.width:] == -5).all())


def test_odd_requests(hip, stream):
    # negative lengths, a need beyond the table, tokens beyond the batch, a table that names no page
    rng = np.random.default_rng(4)
    cached = np.array([-5, 30, 1000, 10, 2 ** 31 - 1, 20, 15, 0])
    new = np.array([3, -2, 1, 6, 1, 9, 1, 2 ** 31 - 1])
    held = np.array([0, 3, 2, 0, 1, 2, 1, 1])
    s = state(rng, 8, 16, cached, new, held, 20, width=5)
    s["table"][5, 1] = s["n_pages"]  # position 16.. of sequence 5
    s["table"][6, 0] = -1
    for t in (s["max_tokens"], 4, 9, 0):
        t = min(t, 1000)
        c = Call(s, stream, max_tokens=t)
        hip.check(hip.mi_hip_page_tables(ctypes.byref(c.args)))
        same(c.got(), ref.page_tables(**dict(s, max_tokens=t)))


def test_no_sequences_and_no_optional_outputs(hip, stream):
    rng = np.random.default_rng(6)
    none = np.zeros(0, np.int64)
    s = state(rng, 0, 16, none, none, none, 5)
    c = Call(s, stream)
    hip.check(hip.mi_hip_page_tables(ctypes.byref(c.args)))
    got = c.got()
    assert got["q_off"].tolist() == [0] and got["refused"].tolist() == [0] and (got["slots"] == -1).all()
    assert got["ring_at"].tolist() == s["ring_at"].tolist()
    s = state(rng, 3, 16, np.array([5, 6, 7]), np.array([1, 2, 30]), np.array([1, 1, 1]), 5)
    c = Call(s, stream)
    c.args.pos = c.args.seq = c.args.n_refused = None
    hip.check(hip.mi_hip_page_tables(ctypes.byref(c.args)))
    want = ref.page_tables(**s)
    got = c.got()
    same({k: got[k] for k in ("slots", "q_off", "n_kv", "table")}, {k: want[k] for k in ("slots", "q_off", "n_kv", "table")})
    assert all((got[k] == -99).all() for k in ("pos", "seq", "refused"))


def test_steps_of_a_server_in_a_graph(hip, stream):
    """A captured step replayed on changing lengths: pages go round the ring, none is lost or dealt twice."""
    import torch
    rng = np.random.default_rng(8)
    n, page = 37, 16
    cached, new = rng.integers(0, 200, n), rng.integers(1, 30, n)
    s = state(rng, n, page, cached, new, -(-cached // page), 160, extra=0, width=40, spare_tokens=3000)
    side = torch.cuda.Stream()
    c = Call(s, side.cuda_stream, in_place=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        hip.check(hip.mi_hip_page_tables(ctypes.byref(c.args)))
    for step in range(40):
        graph.replay()
        want = ref.page_tables(**s)
        got = c.got()
        same(got, want)
        s.update(table=want["table"], ring=want["ring"], ring_at=want["ring_at"], held=want["held"])
        ring = s["ring"][np.arange(*s["ring_at"]) % s["n_pages"]]
        dealt = np.concatenate([s["table"][i, :s["held"][i]] for i in range(n)] + [ring])
        assert np.array_equal(np.sort(dealt), np.arange(s["n_pages"]))
        # some tokens are turned down, some requests end, others begin; a refused one ends
        kept = np.where(want["n_kv"] > 0, np.maximum(want["n_kv"] - rng.integers(0, 8, n), 0), 0)
        kept[rng.random(n) < 0.1] = 0
        s["cached"], s["new"] = np.where(kept < 500, kept, 0), rng.integers(0, 30, n)
        c.inputs["cached"].copy_(dev(s["cached"].astype(np.int32)))
        c.inputs["new"].copy_(dev(s["new"].astype(np.int32)))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("spare", [3, 6000])
def test_long_requests_before_more_sequences(hip, stream, in_place, spare):
    """Requests whose tokens together pass 32 bits stand among the first 1024 sequences of 2100: they, and
    those behind them, do not fit the batch, and the ones before keep their rows. (6000 tokens: the
    tables have several workgroups.)"""
    rng = np.random.default_rng(21)
    n, big = 2100, 2 ** 31 - 1
    cached, new, held = requests(rng, n, 16, 60, 9)
    new[0] = 5
    new[[500, 600, 700, 1023]] = big
    rows = int(new[:500].sum())
    s = state(rng, n, 16, cached, np.where(new == big, 0, new), held, 6000, width=10)
    s.update(new=new, max_tokens=rows + spare)
    c = Call(s, stream, in_place)
    hip.check(hip.mi_hip_page_tables(ctypes.byref(c.args)))
    want, got = ref.page_tables(**s), c.got()
    assert want["n_kv"][:500].any() and (want["slots"][:rows] >= 0).any()
    same(got, want)
