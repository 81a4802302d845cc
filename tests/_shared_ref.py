"""Plain restatements of the operators of rows that share blocks, as a host program does them: forked
tables, a compacted pool, and beam search's selection in 64 bits."""

import math

import numpy as np
import torch


def blocks(tokens, S):
    return -(-tokens // S)


def fork(lengths, parents, new, tables, shares, ring, state, S, max_tokens):
    """(tables, lengths, shares, state, slots, starts, copies, ring, error): the update one row after
    the other.  `new`: a list, or an integer.  error: None, "length" or "blocks"."""
    R, C, N = len(tables), len(tables[0]), len(ring)
    head, count = state
    top = C * S

    def unchanged(error):
        return ([list(t) for t in tables], list(lengths), list(shares), list(state), [-1] * max_tokens, [0] * (R + 1),
                [[-1] * 3] * R, list(ring), error)

    parents = list(range(R)) if parents is None else parents
    if not 0 <= count <= N or any(not -1 <= p < R for p in parents) or any(not 0 <= n <= top for n in lengths):
        return unchanged("length")
    if isinstance(new, int):
        new = [lengths[p] + new if p >= 0 else 0 for p in parents]
    if any(not 0 <= n <= top for n in new):
        return unchanged("length")
    kept = [min(lengths[p], n) if p >= 0 else 0 for p, n in zip(parents, new)]
    owner = {}
    for p in set(parents) - {-1}:
        most = max(k for q, k in zip(parents, kept) if q == p)
        if most % S and shares[tables[p][most // S]] == 0:
            owner[p] = next(r for r in range(R) if parents[r] == p and kept[r] // S == most // S and kept[r] % S)
    was = {}
    for row, n in zip(tables, lengths):
        for b in row[:blocks(n, S)]:
            was[b] = was.get(b, 0) + 1
    out, copies, slots, starts, taken, now = [], [], [], [0], 0, {}
    for r, (p, k, n) in enumerate(zip(parents, kept, new)):
        row = list(tables[p][:k // S]) if k else []
        if k % S and owner.get(p) == r:
            row.append(tables[p][k // S])
        for b in row:
            now[b] = now.get(b, 0) + 1
        if k % S and owner.get(p) != r:
            copies.append([tables[p][k // S], ring[(head + taken) % N], k % S])
        more = blocks(n, S) - len(row)
        row += [ring[(head + taken + i) % N] for i in range(more)]
        taken += more
        slots += [row[i // S] * S + i % S for i in range(k, n)]
        starts.append(len(slots))
        out.append(row + [-1] * (C - len(row)))
    if len(slots) > max_tokens:
        return unchanged("length")
    if taken > count:
        return unchanged("blocks")
    ring = list(ring)
    gone = sorted(set(was) - set(now))
    for i, b in enumerate(gone):
        ring[(head + count + i) % N] = b
    shares = [max(0, now.get(b, 0) - 1) for b in range(N)]
    return (out, list(new), shares, [(head + taken) % N, count - taken + len(gone)],
            slots + [-1] * (max_tokens - len(slots)), starts, copies + [[-1] * 3] * (R - len(copies)), ring, None)


def consistent(tables, lengths, shares, ring, state, S, away=()):
    """Whether rows, shares and ring describe one pool: every block but those in `away` is held or free, the
    shares count the holders, and a partly filled block has one."""
    held = {}
    for row, n in zip(tables, lengths):
        have = blocks(n, S)
        assert all(b == -1 for b in row[have:])
        for b in row[:have]:
            held[b] = held.get(b, 0) + 1
        if n % S:
            assert shares[row[have - 1]] == 0
    free = [ring[(state[0] + i) % len(ring)] for i in range(state[1])]
    assert len(set(free)) == len(free) and not set(free) & set(held)
    assert set(free) | set(held) == set(range(len(ring))) - set(away)
    assert shares == [max(0, held.get(b, 0) - 1) for b in range(len(ring))]


def compact(lengths, tables, shares, ring, state, S):
    """(tables, shares, ring, state, copies) of the compacted pool."""
    N = len(ring)
    held = sorted({b for row, n in zip(tables, lengths) for b in row[:blocks(n, S)]})
    free = sorted(ring[(state[0] + i) % N] for i in range(state[1]))
    pool = sorted(held + free)
    low = set(pool[:len(held)])
    moves = list(zip([b for b in held if b not in low], [b for b in free if b in low]))
    name = {**{b: b for b in held}, **dict(moves)}
    out = [[name[b] for b in row[:blocks(n, S)]] + [-1] * (len(row) - blocks(n, S)) for row, n in zip(tables, lengths)]
    new = [0] * N
    for b in held:
        new[name[b]] = shares[b]
    rest = pool[len(held):]
    return (out, new, rest + [-1] * (N - len(rest)), [0, len(rest)],
            [[a, b, S] for a, b in moves] + [[-1] * 3] * (N // 2 - len(moves)))


def select(logits, scores, beams, count, end=None):
    """(parents, tokens, scores, all_parents, all_tokens, all_scores), the scores in 64 bits, and how far a
    score may be off: its last rounding, half a step of 2^-24 |v| (and of the subtraction, in 64 bits,
    nothing that counts), and 1e-9 for a sum of exponentials that is right to 1e-9 (the logarithm
    of a sum that is off by a share e is off by e)."""
    x = logits.detach().cpu().float().numpy().astype(np.float64)
    s = scores.detach().cpu().numpy().astype(np.float64)
    rows, every, on = x.shape[0], [[], [], []], [[], [], []]
    for r in range(rows // beams):
        found = []
        for row in range(r * beams, (r + 1) * beams):
            top = x[row].max()
            if not np.isfinite(s[row]) or not np.isfinite(top):
                continue
            lse = top + math.log(np.exp(x[row] - top).sum())
            for t in np.argsort(-x[row], kind="stable")[:count].tolist():
                v = s[row] + (x[row, t] - lse)
                if np.isfinite(v) and np.float32(v) > -np.inf:
                    found.append((-v, row, -x[row, t], t))
        found = [(row, t, -v) for v, row, _, t in sorted(found)[:count]]
        go = [c for c in found if c[1] != end][:beams]
        none = (-1, -1, -math.inf)
        for to, part, n in ((every, found, count), (on, go, beams)):
            for k in range(3):
                to[k] += [c[k] for c in part + [none] * (n - len(part))]
    dt = (torch.int32, torch.int32, torch.float64)
    flat = [torch.tensor(v, dtype=t) for v, t in zip(on, dt)]
    return flat + [torch.tensor(v, dtype=t).reshape(-1, count) for v, t in zip(every, dt)]


def score_bound(v):
    return 2.0**-24 * v.abs() + 1e-9
