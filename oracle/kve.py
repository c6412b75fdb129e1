"""Plain fp64 restatements (numpy) of the evicting KV cache and of token sampling, for the tests."""
import numpy as np


def attend(q, k, v, scale):
    """Softmax attention of one query row q [D] over k, v [n, D]: (out [D], weights [n], the sum
    of weights times absolute values [D], the scores' absolute terms' largest sum)."""
    s = (k @ q) * scale
    terms = (np.abs(k) @ np.abs(q)) * abs(scale)
    w = np.exp(s - s.max())
    w /= w.sum()
    return w @ v, w, w @ np.abs(v), float(terms.max())


def kept(weights, positions, budget, sink, recent, there=None):
    """Slots that stay of one (sequence, kv head) and the moves: (sorted kept slots, places, slots
    moved there)."""
    n = len(weights)
    there = np.ones(n, bool) if there is None else there
    newest = positions[there].max() if there.any() else 0
    safe = (positions < sink) | (positions > int(newest) - recent)

    def rank(t):                                   # larger stays
        if not there[t]:
            return (0, 0.0)
        if safe[t]:
            return (3, 0.0)
        return (1, 0.0) if np.isnan(weights[t]) else (2, float(weights[t]) + 0.0)
    order = sorted(range(n), key=lambda t: tuple(-x for x in rank(t)) + (t,))
    stay = set(order[:budget])
    places = [t for t in range(min(budget, n)) if t not in stay]
    moved = [t for t in range(budget, n) if t in stay]
    return sorted(stay), places, moved


def draw(logits, u, T=1.0, k=0, p=1.0, m=0.0):
    """The token of one row of logits (fp64), or -1; none whose e is below 2^-51."""
    x = np.asarray(logits, np.float64)
    if not (x < np.inf).all() or x.max() == -np.inf or not (0 <= T < np.inf):
        return -1
    order = np.argsort(-x, kind="stable")
    if T == 0:
        return int(order[0])
    with np.errstate(over="ignore", under="ignore"):
        e = np.exp((x[order] - x[order[0]]) / T)
    n = len(e) if k <= 0 else min(k, len(e))
    if p < 1.0:
        c = np.cumsum(e[:n])
        n = min(n, max(1, int((c < p * c[-1]).sum()) + 1))
    n = max(1, int((e[:n] >= min(m, 1.0)).sum()))
    back = np.argsort(order[:n], kind="stable")
    e = np.where(e < 2.0 ** -51, 0.0, e)
    c = np.cumsum(e[:n][back])
    i = int(np.searchsorted(c, min(max(u, 0.0), 1.0) * c[-1], side="right"))
    if i >= n:                                     # u = 1: the last token with a share
        i = int(np.nonzero(e[:n][back])[0][-1])
    return int(order[:n][back][i])
