"""Drawing a token from its definition, in 64 bits on the CPU."""
import numpy as np


def kept(l, T=1.0, k=0, p=1.0, min_p=0.0):
    """(indexes of the tokens that stay in the order of the vocabulary, their weights) of one row of logits (64 bits); T > 0."""
    ok = np.flatnonzero(~np.isnan(l) & (l > -np.inf))
    if not len(ok):
        return ok, np.zeros(0)
    order = ok[np.argsort(-l[ok], kind="stable")]
    top = l[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(l[order] == top, 1.0, np.exp((l[order] - top) / T))
    n = len(order)
    if k:
        n = min(n, k)
    if p < 1:
        n = min(n, int(np.searchsorted(np.cumsum(w[:n]), p * w[:n].sum())) + 1)
    n = max(n, 1)
    stay = np.flatnonzero(w[:n] >= min(min_p, 1.0))
    at = np.sort(order[stay])
    back = {i: x for i, x in zip(order[stay], w[stay])}
    return at, np.array([back[i] for i in at])


def token(l, u, T=1.0, k=0, p=1.0, min_p=0.0):
    l = np.asarray(l, np.float64)
    if not (T > 0):
        at = kept(l, 1.0, 1)[0]
        return int(at[0]) if len(at) else -1
    at, w = kept(l, T, k, p, min_p)
    if not len(at):
        return -1
    run = np.cumsum(w)
    i = int(np.searchsorted(run, (u if u > 0 else 0.0) * run[-1], side="right"))
    live = np.flatnonzero(w > 0)
    return int(at[min(i, live[-1])])
