"""Plain 64-bit implementations of sampling, routing and the experts' rows, written from their
definitions with numpy alone, row by row."""
from __future__ import annotations

import numpy as np


def ranked(x):
    """Indices by value descending, equal values by lower index (x holds no NaN)."""
    return np.argsort(-(x + 0.0), kind="stable")


def sample_row(x, q, t, k, p, mp, slack):
    """(tokens that a computation with relative errors up to `slack` may return, log-probability
    of each token) for one row; (None, None) where nothing is open."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    m = x.max()
    if m == -np.inf:
        return None, None
    inv = 1.0 if not t > 0 else 1.0 / t
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        d = np.where(x == m, 0.0, (x - m) * inv)
        w = np.exp(d)
        lp = d - np.log(w.sum())
        order = ranked(x)
        if not t > 0:
            return {int(order[0])}, lp
        n = k if 0 < k < x.size else x.size
        wk = w[order[:n]]
        before = np.concatenate([[0.0], np.cumsum(wk)[:-1]])
        mp = min(max(mp, 0.0), 1.0) if mp == mp else 0.0

        def kept(f):
            ok = (before < p * wk.sum() * f) if p < 1 else np.ones(n, bool)
            ok[0] = True
            ok &= (wk >= min(mp / f, 1.0)) & (x[order[:n]] > -np.inf)
            return order[:n][ok]

        score = w / q.astype(np.float64)
        score = np.where(score >= 0, score, -1.0)
        best = score[kept(1 - slack)].max()
        wide = kept(1 + slack)
        at_least = best * (1 - slack) if best > 0 else best
        return {int(i) for i in wide[score[wide] >= at_least]}, lp


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-x))


def softmax(x):
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        e = np.exp(np.where(x == m, 0.0, x - m))
    return e / e.sum()


def route_row(x, k, score, bias, groups, topk_groups, renorm, scale):
    """(choice of every expert after the groups, chosen experts, weights, scores) of one token."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    s = softmax(x) if score == "softmax" else sigmoid(x)
    c = x.copy() if bias is None else s + bias.astype(np.float64)
    c = np.where((x == -np.inf) | np.isnan(c), -np.inf, c)
    if groups > 1:
        judged = s if (score == "sigmoid" and bias is None) else c
        judged = np.where(c == -np.inf, -np.inf, judged).reshape(groups, -1)
        g = np.empty(groups)
        for i in range(groups):
            best = np.sort(judged[i])[::-1][: 1 if score == "softmax" else 2]
            best = best[best > -np.inf]
            g[i] = best.sum() if best.size else -np.inf
        stay = ranked(g)[:topk_groups]
        mask = np.full(groups, False)
        mask[stay] = True
        c = np.where(np.repeat(mask, x.size // groups), c, -np.inf)
    e = ranked(c)[:k]
    e = np.where(c[e] == -np.inf, -1, e)
    w = np.where(e >= 0, s[e], 0.0)
    w = scale * (w / (w.sum() + 1e-20) if renorm else w)
    return c, e, w, s


def route_grad_row(x, e, g, score, renorm, scale):
    """dL/dx of the weights of chosen experts e for dL/dw = g."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    s = softmax(x) if score == "softmax" else sigmoid(x)
    ok = e >= 0
    sel = np.where(ok, s[e], 0.0)
    big = scale * np.where(ok, g.astype(np.float64), 0.0)
    if renorm:
        total = sel.sum() + 1e-20
        big = (big - (big * sel).sum() / total) / total
    ds = np.zeros_like(s)
    ds[e[ok]] = big[ok]
    if score == "softmax":
        return s * (ds - (ds * s).sum())
    return ds * s * sigmoid(-x)


def order(experts, num):
    """(offsets, order, position) of the assignments, sorted by expert."""
    flat = experts.reshape(-1)
    lists = [np.flatnonzero(flat == e) for e in range(num)]
    offsets = np.concatenate([[0], np.cumsum([len(a) for a in lists])])
    order = np.full(flat.size, -1)
    live = np.concatenate(lists) if lists else np.zeros(0, int)
    order[: live.size] = live
    position = np.full(flat.size, -1)
    position[live] = np.arange(live.size)
    return offsets, order, position.reshape(experts.shape)
