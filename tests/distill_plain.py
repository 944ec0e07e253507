"""Plain 64-bit form of distill_loss and its gradient, row by row."""

import numpy as np


def rows(x, ids, lps, temp=1.0, tail="drop"):
    """x [N, V] float64; (losses [N], gradients [N, V], sizes [N, V]) of
    unweighted rows; sizes: the terms that a gradient is the difference of,
    without those of the teacher, added up."""
    N, V = x.shape
    losses, grads, sizes = np.zeros(N), np.zeros((N, V)), np.zeros((N, V))
    for r in range(N):
        z = x[r] / temp
        m = z.max()
        # m first: m + log of the sum would lose the sum where m is large
        logq = (z - m) - np.log(np.exp(z - m).sum())
        q = np.exp(logq)
        keep = (ids[r] >= 0) & (ids[r] < V)
        i, lp = ids[r][keep].astype(np.int64), lps[r][keep].astype(np.float64)
        if tail == "drop":
            if i.size == 0 or np.isneginf(lp).all():
                continue
            top = lp.max()
            lp = lp - (top + np.log(np.exp(lp - top).sum()))
        p = np.exp(lp)
        some = p != 0
        loss = (p[some] * (lp[some] - logq[i[some]])).sum()
        g, size = q.copy(), q.copy()
        if tail == "bucket":
            outside = np.ones(V, dtype=bool)
            outside[i] = False
            rest = max(0.0, 1.0 - p.sum())
            if outside.any():
                qt = max(q[outside].sum(), 2.0 ** -100)
                if rest > 0:
                    loss += rest * (np.log(rest) - np.log(qt))
                g[outside] = q[outside] * (1.0 - rest / qt)
                size[outside] = q[outside] * (1.0 + rest / qt)
        np.subtract.at(g, i, p)
        losses[r], grads[r], sizes[r] = loss, g / temp, size / temp
    return losses, grads, sizes


def loss(x, ids, lps, temp=1.0, tail="drop", weights=None, reduction="mean", up=None):
    """(loss, gradient, sizes); up: the loss's own gradient, [N] or one value."""
    N = x.shape[0]
    w = np.ones(N) if weights is None else weights.astype(np.float64)
    on = w != 0
    losses, grads, sizes = np.zeros(N), np.zeros_like(x), np.zeros_like(x)
    if on.any():
        losses[on], grads[on], sizes[on] = rows(x[on], ids[on], lps[on], temp, tail)
    losses = losses * w
    if reduction == "none":
        mul = (w * (np.ones(N) if up is None else up))[:, None]
        return losses, grads * mul, sizes * np.abs(mul)
    by = (w.sum() if reduction == "mean" else 1.0)
    by = 1.0 / by if by else 0.0
    mul = w[:, None] * by * (1.0 if up is None else up)
    return losses.sum() * by, grads * mul, sizes * np.abs(mul)
