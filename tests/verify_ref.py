"""Verification of drafted tokens in 64 bits, as the header says it, a sequence at a time."""
import numpy as np


def probabilities(z, temp):
    """softmax(z / temp) of one row, None where it has no distribution"""
    z = z.astype(np.float64)
    if np.isnan(z).any() or (z == np.inf).any() or (z == -np.inf).all():
        return None
    with np.errstate(invalid="ignore"):
        e = np.exp(np.where(z == -np.inf, -np.inf, (z - z.max()) / np.float64(temp)))
    return e / e.sum()


def verified(z, draft, row0, drafted, u, temps, tokens):
    """tokens as they were, with those of the sequences put in; accepted [seqs]"""
    tokens, v = tokens.copy(), z.shape[1]
    accepted = np.zeros(len(row0) - 1, np.int32)
    for b in range(len(accepted)):
        r0, r1 = int(row0[b]), int(row0[b + 1])
        if r0 == r1:
            continue
        temp, stop, follow = np.float32(temps[b]), r1 - 1, -1
        greedy = not temp > 0
        best = lambda p, row: int(np.flatnonzero(z[row] == z[row].max())[0]) if p is not None else -1  # noqa: E731
        for row in range(r0, r1):
            p = probabilities(z[row], 1 if greedy else temp)
            last, x = row == r1 - 1, int(drafted[row])
            there = 0 <= x < v
            q = None if last or greedy else probabilities(draft[row], temp) if draft is not None else np.eye(1, v, x)[0] if there else np.zeros(v)
            if last or p is None:
                ok = False
            elif greedy:
                ok = x == best(p, row)
            else:
                ok = there and q is not None and np.float64(u[row]) * q[x] < p[x]
            if ok:
                continue
            stop = row
            if p is not None and greedy:
                follow = best(p, row)
            elif p is not None:
                r = p if last or q is None else np.maximum(p - q, 0)
                r = r if r.sum() > 0 else p
                run = np.cumsum(r)
                over = np.flatnonzero((run > np.float64(u[r1 - 1]) * run[-1]) & (r > 0))
                follow = int(over[0]) if len(over) else int(np.flatnonzero(r > 0)[-1])
            break
        tokens[r0:stop] = drafted[r0:stop]
        tokens[stop] = follow
        tokens[stop + 1:r1] = -1
        accepted[b] = stop - r0
    return tokens, accepted
