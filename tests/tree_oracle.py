"""Trees of drafted tokens on the host, from their definitions and in 64 bits:
shared by the tests of the mh_kv_tree functions, mh_kv_keep_dev and
mh_verify_dev."""
from __future__ import annotations

import numpy as np

SHAPES = ("any", "chain", "wide", "roots")


def tree(n, shape, rng):
    """Parents of n rows: any earlier row; the row before; all after the first; many that follow the cached tokens."""
    if shape == "chain":
        return list(range(-1, n - 1))
    if shape == "wide":
        return [-1, *[0] * (n - 1)][:n]
    if shape == "roots":
        return [-1 if i == 0 or rng.random() < 0.4 else int(rng.integers(i)) for i in range(n)]
    return [-1, *(int(rng.integers(i)) for i in range(1, n))][:n]


def trees(seqs, shape, rng):
    """Parents of a batch's rows [(len, rows)], one after the other."""
    return np.array([p for _, r in seqs for p in tree(r, shape, rng)], np.int32)


def paths(parent):
    """Of each row of one tree: the rows from the first to it, itself the last. A parent out of range counts as -1."""
    out = []
    for i, p in enumerate(parent):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def seen(base, path, window):
    """The tokens that a row with this path sees, in order; its position is base + len(path) - 1."""
    lo = max(0, base + len(path) - window) if window else 0
    return list(range(lo, base)) + [base + r for r in (path[-window:] if window else path)]


def weights(x, temp):
    """softmax(x / temp) in 64 bits (one-hot of the first maximum for temp <= 0), or None: no probabilities."""
    x = x.astype(np.float64)
    if np.isnan(x).any() or (x == -np.inf).all():
        return None
    if temp <= 0:
        p = np.zeros(len(x))
        p[x.argmax()] = 1.0
        return p
    if (x == np.inf).any():
        return None
    e = np.exp((x - x.max()) / np.float64(np.float32(temp)))
    return e / e.sum()


def verify(logits, parent, token, u, temp, q=None):
    """One sequence, as the header tells it: (kept rows, next token)."""
    V = logits.shape[1]
    path, row = [0], weights(logits[0], temp)
    p = row
    for i in range(1, len(parent)):
        c = int(token[i])
        if parent[i] != path[-1] or p is None or not 0 <= c < V:
            continue
        qq = np.zeros(V) if q is None or temp <= 0 else q[path[-1]].astype(np.float64)
        if q is None or temp <= 0:
            qq[c] = 1.0
        if np.float64(u[i]) * qq[c] < p[c]:
            path.append(i)
            p = row = weights(logits[i], temp)
            continue
        rest = np.maximum(p - qq, 0.0)
        p = rest / rest.sum() if rest.sum() > 0 else rest
    if row is None:
        return path, -1
    if not p.sum() > 0:
        p = row
    run = np.cumsum(p)
    past = np.flatnonzero((run > np.float64(u[0]) * run[-1]) & (p > 0))
    return path, int(past[0]) if len(past) else int(np.flatnonzero(p > 0)[-1])
