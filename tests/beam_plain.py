"""Plain 64-bit forms of top_logprobs, beam_select and beam_reorder that the
tests compare with, written row by row with numpy."""

import numpy as np


def allowed_bits(words, V):
    """[rows, words] packed words (any 32-bit type) -> [rows, V] bool."""
    w = np.ascontiguousarray(words).view(np.uint32)
    return ((w[:, :, None] >> np.arange(32, dtype=np.uint32)) & 1).astype(bool).reshape(w.shape[0], -1)[:, :V]


def pack_bits(allowed):
    rows, V = allowed.shape
    W = (V + 31) // 32
    pad = np.zeros((rows, W * 32), dtype=bool)
    pad[:, :V] = allowed
    return (pad.reshape(rows, W, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32)


def row_lse(z):
    """log sum e^z in 64 bits; NaN if z holds a NaN or +inf, -inf if nothing."""
    if np.isnan(z).any() or np.isposinf(z).any():
        return np.nan
    m = z.max()
    return m if np.isneginf(m) else m + np.log(np.exp(z - m).sum())


def log_softmax(z):
    """z - row_lse(z) without a difference of numbers as large as z: at
    z = 3e38 the logarithm of the sum would be lost in row_lse."""
    m = z.max()
    with np.errstate(invalid="ignore"):
        d = z - m
    return d - np.log(np.exp(d).sum())


def row_best(z, n):
    """Ids of the n best finite values: larger first, then the lower id."""
    order = np.lexsort((np.arange(z.size), -z))
    return [int(i) for i in order[:n] if not np.isneginf(z[i])]


def top_logprobs(x, k, temp=1.0, allowed=None):
    """x [N, V] float64.  (ids, logprobs, lse)."""
    N = x.shape[0]
    ids = np.full((N, k), -1, dtype=np.int32)
    lp = np.full((N, k), -np.inf)
    lse = np.empty(N)
    for r in range(N):
        z = x[r] if allowed is None else np.where(allowed[r], x[r], -np.inf)
        lse[r] = row_lse(z / temp)
        if np.isnan(lse[r]):
            lp[r] = np.nan
            continue
        best = row_best(z, k)
        ids[r, :len(best)] = best
        lp[r, :len(best)] = log_softmax(z / temp)[best]
    return ids, lp, lse


def beam_select(x, scores, n, allowed=None, done=None, eos=-1, lengths=None, alpha=0.0, keep_slots=False):
    """x [B, W, V] float64.  (scores, parents, tokens, lengths, done)."""
    B, W, V = x.shape
    S = np.full((B, n), -np.inf)
    P = np.full((B, n), -1, dtype=np.int32)
    T = np.full((B, n), -1, dtype=np.int32)
    Ln = np.zeros((B, n), dtype=np.int32)
    D = np.zeros((B, n), dtype=bool)
    for b in range(B):
        cand = []  # (-rank, beam, place in the beam's list, total, token, length, done)
        for w in range(W):
            s = float(scores[b, w])
            if np.isneginf(s) or np.isnan(s):
                continue
            base = int(lengths[b, w]) if lengths is not None else 0
            if done is not None and done[b, w]:
                cand.append((-s / max(base, 1) ** alpha, w, 0, s, eos, base, True))
                continue
            z = x[b, w] if allowed is None else np.where(allowed[b * W + w], x[b, w], -np.inf)
            lse = row_lse(z)
            if not np.isfinite(lse):
                continue
            logq = log_softmax(z)
            for j, v in enumerate(row_best(z, n)):
                t = s + logq[v]
                cand.append((-t / max(base + 1, 1) ** alpha, w, j, t, v, base + 1, v == eos))
        cand.sort(key=lambda c: c[:3])
        cand = cand[:n]
        slots = list(range(n))
        if keep_slots:
            where, later = {}, []
            for j, c in enumerate(cand):
                if c[1] in where.values():
                    later.append(j)
                else:
                    where[j] = c[1]
            free = [s for s in range(n) if s not in where.values()]
            later += list(range(len(cand), n))
            for j, s in zip(later, free):
                where[j] = s
            slots = [where[j] for j in range(n)]
        for j, c in enumerate(cand):
            o = slots[j]
            S[b, o], P[b, o], T[b, o], Ln[b, o], D[b, o] = c[3], c[1], c[4], c[5], c[6]
    return S, P, T, Ln, D


def reorder(state, parents, into=None, lengths=None, seq_dim=None):
    """state [B*W, ...]; what lands in `into` (the state itself if None)."""
    B, W = parents.shape
    out = (state if into is None else into).copy()
    for b in range(B):
        for j in range(W):
            p = int(parents[b, j])
            if p < 0 or p >= W:
                p = j
            src = state[b * W + p]
            if lengths is None or seq_dim is None:
                out[b * W + j] = src
            else:
                n = min(max(int(lengths[b, p]), 0), state.shape[seq_dim])
                at = (slice(None),) * (seq_dim - 1) + (slice(0, n),)
                out[b * W + j][at] = src[at]
    return out
