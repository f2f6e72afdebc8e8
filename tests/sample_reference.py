"""Sampling restated in extended precision, one row at a time.

The kernel holds weights to 2^-44 of the largest (one) and adds them exactly, and forms u W and p S in 64 bits: a running sum is
off from its value by at most n (2^-44 + 2^-51) + 2^-52 W, the last for the borders and for weights' own 64-bit arithmetic
(2^-51 of a weight). A choice that lies within twice that of its border may go either way: `choices` gives every token that it may be."""
import numpy as np

LD = np.longdouble


def _kept(x, rule, tol, sign):
    """Ids kept, rising, and their weights; top-p's border moved by sign * tol."""
    t, k, p, least = rule
    n = len(x)
    m = x.max()
    with np.errstate(all="ignore"):
        w = np.where(x == m, LD(1), np.exp(((x.astype(LD) - LD(m)) / LD(np.float32(t)))))
    w = np.where(np.isnan(w) | (x == -np.inf), LD(0), w)
    order = np.lexsort((np.arange(n), -x))
    if 0 < k < n:
        order = order[:k]
    if p < 1:
        ws = w[order]
        before = np.cumsum(ws) - ws
        keep = before < LD(max(np.float32(p), 0)) * ws.sum() + sign * tol
        keep[0] = True
        order = order[keep]
    if least > 0:
        keep = w[order] >= LD(np.float32(least)) * (1 + sign * LD(2) ** -40)
        keep[0] = True
        order = order[keep]
    order = np.sort(order)
    return order, w[order]


def choices(x, rule, u):
    """{id: probabilities} of the tokens that may be drawn from logits x by rule (temperature, top_k, top_p, min_p)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return {-1: [0.0]}
    if not np.float32(rule[0]) > 0:
        return {int(np.argmax(x)): [1.0]}
    tol = 2 * len(x) * (LD(2) ** -44 + LD(2) ** -51)
    found = {}
    for sign in (-1, 0, 1):
        ids, w = _kept(x, rule, tol + LD(2) ** -51 * len(x), sign)
        upto = np.cumsum(w)
        total = upto[-1]
        for off in (-1, 0, 1):
            if np.isnan(u) or u >= 1:
                at = np.nonzero(w > LD(2) ** -45)[0][-1]
            else:
                at = np.searchsorted(upto, max(LD(u), 0) * total + off * (tol + LD(2) ** -51 * total), side="right")
            at = min(max(int(at), int(np.nonzero(w > 0)[0][0])), len(w) - 1)
            found.setdefault(int(ids[at]), []).append(float(w[at] / total))
    return found


def check(ids, prob, x, rules, u, what=""):
    """Every row's token is one that it may be, its probability within a rounding to f32 and the weights' error."""
    for r in range(len(x)):
        may = choices(x[r], rules[r], u[r])
        assert int(ids[r]) in may, (what, r, rules[r], u[r], int(ids[r]), may)
        want = may[int(ids[r])]
        assert any(abs(float(prob[r]) - p) <= p * 2.0 ** -23 + len(x[r]) * 2.0 ** -42 for p in want), (
            what, r, rules[r], u[r], float(prob[r]), want)
