"""Plain 64-bit restatement of the draw from a row of logits, for the tests."""
import numpy as np


def draw(x, u, t=1.0, k=0, p=1.0, least=0.0):
    """(id, its share, how close the draw and the rules came to the next word, of all weights) of one row."""
    x = np.asarray(x, np.float64)
    t, k, p, least, u = float(t), int(k), float(p), float(least), float(u)
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return -1, 0.0, 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    if not t > 0:
        return int(order[0]), 1.0, 1.0
    with np.errstate(over="ignore"):
        w = np.exp((x[order] - x[order[0]]) / t)
    n, close = len(x), 1.0
    if k > 0:
        n = min(n, k)
    if p < 1:
        upto = np.cumsum(w[:n].astype(np.longdouble))
        goal = np.longdouble(p) * upto[-1]
        before = np.concatenate(([0], upto[:-1]))
        close = min(close, float(np.abs(before[1:] - goal).min() / upto[-1]) if n > 1 else 1.0)
        n = max(1, int((before < goal).sum()))
    if least > 0:
        below = w[:n][x[order[:n]] < x[order[0]]]   # (those that share the largest weigh 1 exactly)
        close = min(close, float(np.abs(below / least - 1).min()) if len(below) else 1.0)
        n = max(1, int((w[:n] >= least).sum()))
    kept = np.zeros(len(x), np.longdouble)
    kept[order[:n]] = w[:n]
    upto = np.cumsum(kept)
    u = 0.0 if not u > 0 else min(u, 1.0)
    goal = u * upto[-1]
    hit = np.nonzero(upto > goal)[0]
    i = int(hit[0]) if len(hit) else int(np.nonzero(kept)[0][-1])
    if 0 < u < 1:
        close = min(close, float(min(upto[i] - goal, goal - (upto[i] - kept[i])) / upto[-1]))
    return i, float(kept[i] / upto[-1]), close
