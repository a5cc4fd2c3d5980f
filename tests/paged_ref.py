"""Plain 64-bit forms of the operators over a paged cache, for their tests."""
import numpy as np


def page_tables(page, n_pages, max_pages, max_tokens, cached, new, held, table, ring, ring_at):
    """What mi_hip_page_tables writes, sequence by sequence."""
    table, ring = table.copy(), ring.copy()
    head, tail = int(ring_at[0]), int(ring_at[1])
    free, taken, q = tail - head, 0, 0
    held_out, n_kv, q_off, refused = held.copy(), [], [0], 0
    slots, pos, seq = np.full(max_tokens, -1), np.zeros(max_tokens, int), np.full(max_tokens, -1)
    old = ring.copy()
    for i in range(len(cached)):
        c, f = max(int(cached[i]), 0), max(int(new[i]), 0)
        need = -(-(c + f) // page)
        start, q = q, q + f
        take = max(0, need - int(held[i]))
        ok = need <= max_pages and q <= max_tokens
        if ok:
            taken += take
            ok = take == 0 or taken <= free
        if ok:
            for k in range(take):
                table[i, held[i] + k] = old[(head + taken - take + k) % n_pages]
            for k in range(need, int(held[i])):
                ring[tail % n_pages] = table[i, k]
                tail += 1
            held_out[i] = need
        refused += not ok
        n_kv.append(c + f if ok else 0)
        q_off.append(min(q, max_tokens))
        for j in range(start, min(q, max_tokens)):
            seq[j], pos[j] = i, c + j - start
            if ok:
                e = table[i, pos[j] // page]
                slots[j] = e * page + pos[j] % page if 0 <= e < n_pages else -1
    granted = sum(max(0, int(held_out[i]) - int(held[i])) for i in range(len(cached)))
    head += granted
    laps = head // n_pages * n_pages
    return dict(held=held_out, table=table, ring=ring, ring_at=np.array([head - laps, tail - laps]), n_kv=np.array(n_kv, int),
                q_off=np.array(q_off), slots=slots, pos=pos, seq=seq, refused=np.array([refused]))


def weights(x, temperature):
    """exp((x - max) / T) of a row of logits, one at the lowest of the largest for T = 0; None for a row
    without a distribution."""
    x = x.astype(np.float64)
    if not (x < np.inf).all() or x.max() == -np.inf:
        return None
    if temperature > 0:
        return np.exp((x - x.max()) / float(temperature))
    w = np.zeros(len(x))
    w[int(x.argmax())] = 1.0
    return w


def verify(logits, token, parent, draft, temperature, u, max_path):
    """(path, tokens) of one sequence of nodes, as mi_hip_verify_draft gives them (without the -1s
    behind them), and the least distance of a test or of the draw from its border."""
    n, vocab = logits.shape
    u = np.clip(u.astype(np.float64), 0.0, 1.0 - 2.0 ** -24)
    w = [weights(x, temperature) for x in logits]
    p = [None if x is None else x / x.sum() for x in w]
    cur, path, tokens, down, left, margin = 0, [0], [], [], 1.0, 1.0
    for c in range(1, n):
        if len(path) == max_path:
            break
        if (c - 1 if parent is None else int(parent[c])) != cur:
            continue
        t = int(token[c])
        known = 0 <= t < vocab and p[cur] is not None and t not in [int(token[e]) for e in down]
        pc = p[cur][t] if known else 0.0
        bar = u[c] * (left if draft is None else float(draft[c, t]) if 0 <= t < vocab else 1.0)
        if pc > 0.0:
            margin = min(margin, abs(bar - pc))
        if bar < pc:
            tokens.append(t)
            path.append(c)
            cur, down, left = c, [], 1.0
        else:
            left -= pc
            down.append(c)
    if len(path) == max_path:
        down = []
    if p[cur] is None:
        return path, tokens + [-1], margin
    if draft is not None and down:
        rest = np.maximum(p[cur] - draft[down[0]].astype(np.float64), 0.0)
    else:
        rest = w[cur].copy()
        for e in down:
            if 0 <= int(token[e]) < vocab:
                rest[int(token[e])] = 0.0
    cum = np.cumsum(rest)
    target = u[0] * cum[-1]
    if cum[-1] == 0.0:
        return path, tokens + [-1], margin
    steps = cum[np.concatenate([[True], np.diff(cum) > 0])]
    margin = min(margin, np.abs(steps - target)[steps > 0].min() / cum[-1])
    above = np.nonzero(cum > target)[0]
    return path, tokens + [int(above[0]) if len(above) else int(np.nonzero(rest)[0][-1])], margin
