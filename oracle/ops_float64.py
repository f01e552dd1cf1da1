"""The operators on row tables and score rows (vectordb_amd.ops) from their definitions, in float64 NumPy, one row after the
other.  Test infrastructure only."""

import math

import numpy as np

UNIT = 2.0 ** -24                      # half a step of float32, relative


def lookup(table, rows, scale):
    table = np.asarray(table, np.float64)
    out = np.zeros((len(rows), table.shape[1]))
    for i, r in enumerate(rows):
        if 0 <= r < len(table):
            out[i] = scale * table[r]
    return out


def lookup_grad(grad, rows, n_rows, scale):
    """(sums, sums of magnitudes, number of terms) per table row"""
    grad = np.asarray(grad, np.float64)
    out, mag, cnt = np.zeros((n_rows, grad.shape[1])), np.zeros((n_rows, grad.shape[1])), np.zeros(n_rows, np.int64)
    ok = (rows >= 0) & (rows < n_rows)
    np.add.at(out, rows[ok], scale * grad[ok])
    np.add.at(mag, rows[ok], abs(scale) * np.abs(grad[ok]))
    np.add.at(cnt, rows[ok], 1)
    return out, mag, cnt


def teacher_probabilities(t, rows, vocab, tau, lse=None):
    """p_j and log p_j of one list (0 and -inf where unfilled)."""
    filled = (rows >= 0) & (rows < vocab) & (t != -np.inf)
    x = np.where(filled, t / tau, -np.inf)
    if not filled.any():
        return np.zeros(len(t)), np.full(len(t), -np.inf)
    with np.errstate(over="ignore"):
        logp = x - (lse if lse is not None else np.max(x) + math.log(np.sum(np.exp(x - np.max(x)))))
    return np.exp(logp), logp


def distill_row(z, t, rows, tau, lse=None):
    """loss and gradient (for an upstream gradient of 1) of one row, with the quantities its error bounds need."""
    z = np.asarray(z, np.float64)
    vocab = len(z)
    p, logp = teacher_probabilities(np.asarray(t, np.float64), rows, vocab, tau, lse)
    mass = p.sum()
    top = z.max()
    base = top if top > -np.inf else 0.0
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        d = (z - base) / tau                                   # <= 0
        w = np.exp(d)
        s = w.sum()
        logs = np.log(s)
        q = w / s if s > 0 else np.zeros(vocab)
        loss, target = 0.0, np.zeros(vocab)
        for j in range(len(p)):
            if p[j] > 0:
                loss += p[j] * (logp[j] - (d[rows[j]] - logs))
                target[rows[j]] += p[j]
    out = {"p": p, "logp": logp, "mass": mass, "q": q, "d": d, "s": s, "logs": logs, "top": top, "target": target,
           "loss": tau * tau * loss, "grad": tau * (mass * q - target)}
    if mass == 0:
        out["loss"], out["grad"] = 0.0, np.zeros(vocab)
    return out


def sample_row(z, u, tau, top_k=0, top_p=1.0, min_p=0.0, allowed=None):
    """(row, log-probability) drawn from one score row."""
    z = np.asarray(z, np.float64)
    can = ~np.isnan(z) & (z != -np.inf)
    if allowed is not None:
        can &= allowed
    place = np.flatnonzero(can)
    if len(place) == 0:
        return -1, -np.inf
    place = place[np.argsort(-z[place], kind="stable")]
    best = z[place[0]]
    if not tau > 0:
        place, tau = place[:1], 1.0
    if top_k > 0:
        place = place[:top_k]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(z[place] == best, 1.0, np.exp((z[place] - best) / tau))
    w = np.where(w >= 2.0 ** -40, w, 0.0)                       # NaN too
    n = len(place)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int(np.sum(before < top_p * w.sum())))
    if min_p > 0:
        n = min(n, int(np.sum(w >= min(min_p, 1.0))))
    order = np.argsort(place[:n], kind="stable")
    place, w = place[:n][order], w[:n][order]
    reach = np.cumsum(w)
    j = int(np.searchsorted(reach, u * reach[-1], side="right"))
    j = min(j, int(np.flatnonzero(w)[-1]))
    return int(place[j]), math.log(w[j] / reach[-1])
