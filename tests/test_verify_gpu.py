"""Verification of drafted tokens (mi_hip_verify_draft) against 64 bits: whole numbers, equal where no test
and no draw is closer to its border than the two forms' sums may differ (n_vocab roundings of 2^-53)."""
import ctypes

import numpy as np
import pytest

import mi_hip_attn as mh
import paged_ref as ref
from test_kv8_gpu import dev

pytestmark = pytest.mark.gpu


def softmax(x):
    e = np.exp(x.astype(np.float64) - x.max())
    return e / e.sum()


def draft_rows(rng, logits, off, noise):
    """A draft model's probabilities and a token drawn from each, for chains."""
    draft = np.full(logits.shape, np.nan, np.float32)  # (rows of node 0 are not read)
    token = np.zeros(len(logits), np.int32)
    for i in range(len(off) - 1):
        for r in range(off[i] + 1, off[i + 1]):
            guess = softmax(logits[r - 1] + noise * rng.standard_normal(logits.shape[1]))
            draft[r] = guess
            token[r] = rng.choice(len(guess), p=guess)
    return draft, token


def likely(rng, logits, off, parent, spread):
    """Likely tokens of each node's parent's row."""
    token = np.zeros(len(logits), np.int32)
    for i in range(len(off) - 1):
        for c in range(1, off[i + 1] - off[i]):
            v = c - 1 if parent is None else parent[off[i] + c]
            token[off[i] + c] = np.argsort(-logits[off[i] + v])[int(rng.integers(0, spread))]
    return token


class Case:
    def __init__(self, logits, off, token, u, parent=None, draft=None, temperature=None, max_path=None, pad=0):
        self.logits, self.off, self.token, self.u = logits, off, token, u
        self.parent, self.draft, self.temperature = parent, draft, temperature
        self.n = len(off) - 1
        self.max_path = max(1, int(np.diff(off).max(initial=1))) if max_path is None else max_path
        self.pad = pad

    def call(self, hip, stream, ws=None):
        import torch
        rows, vocab = self.logits.shape
        wide = torch.full((rows, vocab + self.pad), float("nan"), device="cuda")
        wide[:, :vocab] = dev(self.logits)
        dwide = None
        if self.draft is not None:
            dwide = torch.full((rows, vocab + 2 * self.pad), float("nan"), device="cuda")
            dwide[:, :vocab] = dev(self.draft)
            dwide = dwide[:, :vocab]
        i32 = lambda x: None if x is None else dev(np.asarray(x, np.int32))
        self.n_path = torch.full((self.n,), -9, dtype=torch.int32, device="cuda")
        self.path = torch.full((self.n, self.max_path + 1), -9, dtype=torch.int32, device="cuda")
        self.tokens = torch.full((self.n, self.max_path + 2), -9, dtype=torch.int32, device="cuda")
        self.keep = [wide, dwide, i32(self.off), i32(self.token), dev(self.u), i32(self.parent),
                     None if self.temperature is None else dev(np.asarray(self.temperature, np.float32))]
        k = self.keep
        return mh.verify_args(wide[:, :vocab], k[2], k[3], k[4], self.n_path, self.path[:, :self.max_path],
                              self.tokens[:, :self.max_path], stream, parent=k[5], draft=dwide, temperature=k[6], ws=ws)

    def run(self, hip, stream, ws=None):
        import torch
        a = self.call(hip, stream, ws)
        hip.check(hip.mi_hip_verify_draft(ctypes.byref(a)))
        torch.cuda.synchronize()
        return self.results()

    def results(self):
        path, tokens = self.path.cpu().numpy(), self.tokens.cpu().numpy()
        assert (path[:, self.max_path:] == -9).all() and (tokens[:, self.max_path:] == -9).all()
        return self.n_path.cpu().numpy(), path[:, :self.max_path], tokens[:, :self.max_path]

    def want(self, i):
        s = slice(self.off[i], self.off[i + 1])
        t = 1.0 if self.temperature is None else self.temperature[i]
        return ref.verify(self.logits[s], self.token[s], None if self.parent is None else self.parent[s],
                          None if self.draft is None else self.draft[s], t, self.u[s], self.max_path)

    def check(self, got):
        n_path, path, tokens = got
        close = 0
        for i in range(self.n):
            if self.off[i + 1] == self.off[i]:
                assert n_path[i] == 0 and (path[i] == -1).all() and (tokens[i] == -1).all()
                continue
            p, t, margin = self.want(i)
            if margin < self.logits.shape[1] * 2.0 ** -53:
                close += 1  # (either side is right)
                continue
            assert n_path[i] == len(p), (i, n_path[i], p)
            assert path[i].tolist() == p + [-1] * (self.max_path - len(p)), i
            assert tokens[i].tolist() == t + [-1] * (self.max_path - len(t)), (i, tokens[i], t)
        return close


def offsets(rng, n, most, least=1):
    return np.concatenate([[0], np.cumsum(rng.integers(least, most + 1, n))])


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4097, 32000, 151936])
@pytest.mark.parametrize("kind", ["certain", "draft", "tree"])
def test_against_64_bits(hip, stream, vocab, kind):
    rng = np.random.default_rng([vocab, len(kind)])
    n = 12 if vocab > 20000 else 40
    off = offsets(rng, n, 8 if kind != "tree" else 20, 0 if kind == "certain" else 1)
    rows = int(off[-1])
    logits = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    parent = draft = None
    if kind == "draft":
        draft, token = draft_rows(rng, logits, off, 1.0)
    else:
        if kind == "tree":
            parent = np.concatenate([[0] + [int(rng.integers(max(0, c - 4), c)) for c in range(1, k)] for k in np.diff(off)])
        token = likely(rng, logits, off, parent, min(vocab, 3))
    u = rng.random(rows).astype(np.float32)
    temperature = rng.choice([0.0, 0.3, 0.7, 1.0, 1.5], n).astype(np.float32)
    c = Case(logits, off, token, u, parent, draft, temperature, pad=3)
    got = c.run(hip, stream)
    assert c.check(got) <= n // 4
    again = c.run(hip, stream)
    assert all(np.array_equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("kind", ["certain", "draft", "tree"])
def test_long_paths(hip, stream, kind):
    # sharper rows: paths of every length
    rng = np.random.default_rng(len(kind))
    vocab, n = 5000, 60
    off = offsets(rng, n, 12, 2)
    rows = int(off[-1])
    logits = (rng.standard_normal((rows, vocab)) * 8).astype(np.float32)
    parent = draft = None
    if kind == "draft":
        draft, token = draft_rows(rng, logits, off, 1.0)
    else:
        if kind == "tree":
            parent = np.concatenate([[0] + [int(rng.integers(max(0, c - 3), c)) for c in range(1, k)] for k in np.diff(off)])
        token = likely(rng, logits, off, parent, 2)
    c = Case(logits, off, token, rng.random(rows).astype(np.float32), parent, draft, pad=1)
    got = c.run(hip, stream)
    assert c.check(got) == 0
    assert len(set(got[0].tolist())) >= 4


@pytest.mark.parametrize("kind", ["certain", "draft"])
def test_distribution(hip, stream, kind):
    """The tokens that come out are the target's: the first one's counts over 20000 sequences against the
    exact probabilities. A count is binomial; six standard deviations are passed with 2e-9 per token."""
    rng = np.random.default_rng(5)
    vocab, n = 11, 20000
    row = (rng.standard_normal((2, vocab)) * 1.5).astype(np.float32)
    logits = np.tile(row, (n, 1))
    off = 2 * np.arange(n + 1)
    q = softmax(row[0] + 1.2 * rng.standard_normal(vocab)).astype(np.float32)
    draft = token = None
    token = np.zeros(2 * n, np.int32)
    if kind == "draft":
        q = (q.astype(np.float64) / q.astype(np.float64).sum())
        token[1::2] = rng.choice(vocab, n, p=q)
        draft = np.tile(q.astype(np.float32), (2 * n, 1))
    else:
        token[1::2] = int(row[0].argmax())
    c = Case(logits, off, token, rng.random(2 * n).astype(np.float32), draft=draft)
    n_path, _, tokens = c.run(hip, stream)
    p = softmax(row[0])
    counts = np.bincount(tokens[:, 0], minlength=vocab)
    assert np.all(np.abs(counts - n * p) <= 6 * np.sqrt(n * p * (1 - p)) + 1)
    taken = np.minimum(p, q).sum() if kind == "draft" else p.max()
    assert abs((n_path == 2).sum() - n * taken) <= 6 * np.sqrt(n * taken * (1 - taken))
    second = tokens[n_path == 2, 1]
    p2, m = softmax(row[1]), len(second)
    assert np.all(np.abs(np.bincount(second, minlength=vocab) - m * p2) <= 6 * np.sqrt(m * p2 * (1 - p2)) + 1)


def test_equal_logits_are_equal_tokens(hip, stream):
    # weights of exactly one: token floor(u V), for every u, the borders among them
    vocab = 4096
    u = np.concatenate([np.arange(64) / 64, np.arange(1, 64) / 64 - 2.0 ** -24, [0.0, 1.0 - 2.0 ** -24, 0.25]]).astype(np.float32)
    n = len(u)
    c = Case(np.full((n, vocab), -3.25, np.float32), np.arange(n + 1), np.zeros(n, np.int32), u)
    _, _, tokens = c.run(hip, stream)
    assert tokens[:, 0].tolist() == np.floor(u.astype(np.float64) * vocab).astype(int).tolist()


def test_greedy(hip, stream):
    # ties go to the lowest token, -0 equals 0; a child is accepted if it is that token
    vocab = 5000
    x = np.full((6, vocab), -1.0, np.float32)
    x[0, [77, 4000]] = 5.0
    x[1, 3] = 0.0
    x[1, 2] = -0.0
    x[2, 4999] = np.float32(1e30)
    x[3:] = x[:3]
    token = np.array([0, 77, 2, 0, 4000, 2], np.int32)
    for u in (0.0, 0.5, 1.0):
        c = Case(x, np.array([0, 3, 6]), token, np.full(6, u, np.float32), temperature=np.zeros(2, np.float32))
        n_path, path, tokens = c.run(hip, stream)
        assert n_path.tolist() == [3, 1] and tokens.tolist() == [[77, 2, 4999], [77, -1, -1]]
        assert path.tolist() == [[0, 1, 2], [0, -1, -1]]


def test_numbers_at_and_outside_their_range(hip, stream):
    # u of 0, 1, above, below and NaN: clamped; u 0 draws the first token with a weight
    vocab = 100
    x = np.zeros((6, vocab), np.float32)
    x[:, :7] = -np.inf
    x[:, 90:] = -np.inf
    u = np.array([0.0, 1.0, 7.0, -2.0, np.nan, np.inf], np.float32)
    c = Case(x, np.arange(7), np.zeros(6, np.int32), u)
    _, _, tokens = c.run(hip, stream)
    got = tokens[:, 0].tolist()
    assert got[0] == 7 and got[1] == got[2] == got[5] == 89 and got[3] == 7 and got[4] in range(7, 90)


def test_rows_without_a_distribution(hip, stream):
    vocab = 3000
    rng = np.random.default_rng(1)
    x = rng.standard_normal((10, vocab)).astype(np.float32)
    x[0] = -np.inf
    x[2, 1500] = np.nan
    x[4, 0] = np.inf
    x[7] = np.nan
    off, token = np.array([0, 2, 4, 6, 8, 10]), np.zeros(10, np.int32)
    token[[1, 3, 5, 7, 9]] = [5, 6, 0, 8, int(x[8].argmax())]
    u = np.zeros(10, np.float32)
    c = Case(x, off, token, u)
    n_path, path, tokens = c.run(hip, stream)
    # rows 0, 2 and 4 accept nothing and draw nothing; 6 accepts (u = 0) and then has no token from row 7
    assert n_path.tolist() == [1, 1, 1, 2, 2]
    assert tokens.tolist()[:3] == [[-1, -1]] * 3 and tokens[3].tolist() == [8, -1]
    assert tokens[4, 0] == token[9] and tokens[4, 1] == 0


def test_tokens_and_parents_that_are_none(hip, stream):
    # tokens outside the vocabulary are turned down; a node whose parent is not before it has none
    rng = np.random.default_rng(2)
    vocab = 500
    x = rng.standard_normal((16, vocab)).astype(np.float32)
    best = x.argmax(1)
    token = np.array([0, vocab, best[0], best[2], 0, -1, 2 ** 31 - 1, best[4], 0, best[8], best[8], best[8], 0, 1, 2, 3], np.int32)
    parent = np.array([0, 0, 0, 2, 0, 0, 0, 0, 5, 1, 2, 0, -1, 1, 7, 0], np.int32)
    off = np.array([0, 4, 8, 12, 16])
    u = np.zeros(16, np.float32)
    c = Case(x, off, token, u, parent=parent)
    got = c.run(hip, stream)
    c.check(got)
    assert got[0].tolist()[:3] == [3, 2, 2] and got[1][0].tolist() == [0, 2, 3, -1] and got[1][1].tolist()[:2] == [0, 3]
    assert got[1][2].tolist()[:2] == [0, 3]
    # the same token again among siblings is never accepted once turned down
    sib = np.array([0, 0, 0, 0], np.int32)
    tok = np.array([0, 9, 9, 9], np.int32)
    u = np.array([0.3, 1.0, 0.0, 0.0], np.float32)
    c = Case(x[:4], np.array([0, 4]), tok, u, parent=sib)
    got = c.run(hip, stream)
    assert c.check(got) == 0 and got[0][0] == 1 and got[2][0, 0] != 9


def test_paths_end_where_their_list_does(hip, stream):
    rng = np.random.default_rng(3)
    vocab = 700
    x = (rng.standard_normal((24, vocab)) * 3).astype(np.float32)
    off = np.array([0, 6, 12, 18, 24])
    token = likely(rng, x, off, None, 1)
    u = np.zeros(24, np.float32)  # everything is accepted
    u[off[:-1]] = rng.random(4)
    for most in (1, 3, 6, 9):
        c = Case(x, off, token, u, max_path=most)
        got = c.run(hip, stream)
        assert c.check(got) == 0 and (got[0] == min(most, 6)).all()


def test_many_nodes_and_rows_of_no_sequence(hip, stream):
    # a sequence of more than 1024 nodes counts its first 1024; rows before and behind belong to nobody
    rng = np.random.default_rng(4)
    vocab, n = 64, 1100
    x = (rng.standard_normal((n + 5, vocab)) * 6).astype(np.float32)
    off = np.array([2, 2 + n])
    token = likely(rng, x, off, None, 1)
    u = np.zeros(n + 5, np.float32)
    u[2] = 0.4
    c = Case(x, off, token, u, max_path=n)
    n_path, path, tokens = c.run(hip, stream)
    assert n_path[0] == 1024 and path[0, :1024].tolist() == list(range(1024)) and (path[0, 1024:] == -1).all()
    last = np.cumsum(softmax(x[2 + 1023]))
    assert tokens[0, 1023] == np.nonzero(last > np.float64(np.float32(0.4)))[0][0]
    # offsets that no batch has
    c = Case(x, np.array([-4, 3, 2 ** 31 - 1]), token, u, max_path=5)
    c.n = 2
    c.run(hip, stream)


def test_peaked_residuals(hip, stream):
    """A draft that is almost the target, and certain tokens that have almost all of its mass: what is left
    is far below the sums' roundings, but not zero."""
    rng = np.random.default_rng(6)
    vocab = 9000
    x = np.zeros((8, vocab), np.float32)
    x[:, 4321] = 40.0  # the others together: 9000 exp(-40)
    token = np.array([0, 4321] * 4, np.int32)
    u = np.array([0.1, 1.0, 0.5, 1.0, 0.9, 1.0, 0.0, 1.0], np.float32)
    c = Case(x, np.array([0, 2, 4, 6, 8]), token, u)
    n_path, _, tokens = c.run(hip, stream)
    # (1 - 2^-24 is below the token's share: accepted, then drawn from the next row)
    assert (n_path == 2).all()
    parent = np.zeros(8, np.int32)
    x = np.zeros((3, vocab), np.float32)
    x[0, 4321] = 12.0
    c = Case(x, np.array([0, 3]), np.array([0, 4321, 17], np.int32), np.array([0.5, 0.99999, 0.9999], np.float32), parent=parent[:3])
    got = c.run(hip, stream)
    # (half of 8998 equal weights: a border, the 4500th of them or, if the sums round down, the one before)
    assert got[0][0] == 1 and got[2][0, 0] in (4500, 4501)


def test_graph_and_streams(hip, stream):
    import torch
    rng = np.random.default_rng(7)
    vocab = 20000
    off = offsets(rng, 9, 6)
    x = (rng.standard_normal((int(off[-1]), vocab)) * 3).astype(np.float32)
    draft, token = draft_rows(rng, x, off, 1.0)
    c = Case(x, off, token, rng.random(len(x)).astype(np.float32), draft=draft)
    want = c.run(hip, stream)
    c.check(want)
    side = torch.cuda.Stream()
    ws = hip.workspace_create(2, 4, 64)
    with torch.cuda.stream(side):
        a = c.call(hip, side.cuda_stream, ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        hip.check(hip.mi_hip_verify_draft(ctypes.byref(a)))
    for step in range(4):
        c.u = rng.random(len(x)).astype(np.float32)
        c.keep[4].copy_(dev(c.u))
        g.replay()
        torch.cuda.synchronize()
        c.check(c.results())
    hip.check(hip.mi_hip_workspace_destroy(ws))


def test_no_sequences_and_no_rows(hip, stream):
    import torch
    x = np.zeros((0, 100), np.float32)
    c = Case(x, np.array([0, 0, 0]), np.zeros(0, np.int32), np.zeros(0, np.float32), max_path=3)
    n_path, path, tokens = c.run(hip, stream)
    assert n_path.tolist() == [0, 0] and (path == -1).all() and (tokens == -1).all()
    a = c.call(hip, stream)
    a.n_seq = 0
    assert hip.mi_hip_verify_draft(ctypes.byref(a)) == 0
    torch.cuda.synchronize()


def test_rows_beyond_the_workspace(hip, stream):
    a = mh.VerifyArgs()
    c = Case(np.zeros((1, 100), np.float32), np.array([0, 1]), np.zeros(1, np.int32), np.zeros(1, np.float32))
    a = c.call(hip, stream)
    a.n_rows = 2 ** 31 - 1
    assert hip.mi_hip_verify_draft(ctypes.byref(a)) == 5 and "workspace" in hip.last_error()


@pytest.mark.parametrize("vocab", [500, 9000, 60000])
@pytest.mark.parametrize("kind", ["chain", "tree", "draft"])
def test_tokens_outside_the_vocabulary_leave_it_whole(hip, stream, vocab, kind):
    """Drafted tokens that are no tokens are turned down, and nothing is missing from what the next one is drawn
    from: neither the vocabulary's first tokens nor its last ones."""
    rng = np.random.default_rng([vocab, len(kind)])
    none = np.array([-1, -2, -2047, -4097, -2 ** 31, vocab, vocab + 1, 2 ** 31 - 1])
    n, nodes = 64, 4 if kind == "tree" else 2
    off = np.arange(n + 1) * nodes
    logits = rng.standard_normal((n * nodes, vocab)).astype(np.float32)
    token = rng.choice(none, n * nodes)
    parent = draft = None
    if kind == "tree":
        parent = np.zeros(n * nodes, np.int32)
        token[3::4] = logits[0::4].argmax(1)  # one that is, among those that are not
    if kind == "draft":
        draft, _ = draft_rows(rng, logits, off, 1.0)
    u = rng.random(n * nodes).astype(np.float32)
    u[0::nodes] = (np.arange(n) + 0.5) / n  # draws from all of the vocabulary
    c = Case(logits, off, token, u, parent, draft)
    got = c.run(hip, stream)
    assert c.check(got) <= 1
    assert (got[2][:, 0] >= 0).all() and got[2][:, 0].min() < vocab // 8 and got[2][:, 0].max() >= vocab - vocab // 8


@pytest.mark.parametrize("vocab,rows", [(1, 1000000), (4097, 250000)])
def test_scratch_that_the_header_gives(hip, stream, vocab, rows):
    """A call of the header's size is taken by the 17 MB of parts of a workspace for heads of 64, of which it
    asks for most; one of four times the rows is refused."""
    import torch
    n, c = 1000, -(-vocab // 2048)
    assert 12e6 < 16 * c * rows + (8 * c + 40) * n < 17e6
    ws = hip.workspace_create(2, 14, 64)
    i32 = lambda *s: torch.full(s, -9, dtype=torch.int32, device="cuda")
    # every u is 0, so every node is accepted as far as the paths go
    logits, u = torch.zeros(rows, vocab, device="cuda"), torch.zeros(rows, device="cuda")
    token, off = torch.zeros(rows, dtype=torch.int32, device="cuda"), dev((np.arange(n + 1) * (rows // n)).astype(np.int32))
    n_path, path, tokens = i32(n), i32(n, 3), i32(n, 3)
    a = mh.verify_args(logits, off, token, u, n_path, path, tokens, stream, ws=ws)
    a.n_rows = 4 * rows
    assert hip.mi_hip_verify_draft(ctypes.byref(a)) == 5 and "parts" in hip.last_error()
    torch.cuda.synchronize()
    assert bool((n_path == -9).all())
    a.n_rows = rows
    hip.check(hip.mi_hip_verify_draft(ctypes.byref(a)))
    torch.cuda.synchronize()
    assert bool((n_path == 3).all()) and bool((tokens == 0).all())
    assert bool((path == torch.arange(3, device="cuda")).all())
    hip.check(hip.mi_hip_workspace_destroy(ws))
