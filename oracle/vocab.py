"""CPU oracle for the operators on vocabulary rows (numpy, float64): a teacher's
top logits, the cross-entropy against them, token sampling, and the scaled
embedding with its gradient.

TEST INFRASTRUCTURE. Only ``tests/`` imports this module, and only as the
checker. Each function follows the definition in include/mtp_glora_amd.h row by
row; tests/test_oracle_vocab.py pins them against other formulations.
"""
from __future__ import annotations

import numpy as np


def order(row):
    """Columns of a row in order: value descending, column ascending, NaN last."""
    row = np.asarray(row, np.float64)
    key = np.where(np.isnan(row), -np.inf, row)
    # NaN behind -inf, else by value; the sort is stable
    return np.lexsort((np.arange(len(row)), -key, np.isnan(row)))


def logsumexp(row):
    row = np.asarray(row, np.float64)
    m = row.max()
    if np.isnan(m) or np.isinf(m):
        return m
    return m + np.log(np.exp(row - m).sum())


def top_logits(x, k, temperature=1.0):
    """values, ids, lse of rows x [N, V]."""
    x = np.asarray(x, np.float64)
    ids = np.stack([order(r)[:k] for r in x]).astype(np.int64)
    return np.take_along_axis(x, ids, 1), ids, np.array([logsumexp(r / temperature) for r in x])


def teacher_weights(values, ids, V, lse=None, temperature=1.0):
    """q [N, K]: 0 for what does not count."""
    s = np.asarray(values, np.float64) / temperature
    ids = np.asarray(ids)
    s = np.where((ids >= 0) & (ids < V), s, -np.inf)
    q = np.zeros_like(s)
    for r in range(len(s)):
        norm = logsumexp(s[r]) if lse is None else float(lse[r])
        if norm != -np.inf:
            q[r] = np.where(s[r] == -np.inf, 0.0, np.exp(s[r] - norm))
    return q


def top_ce(x, values, ids, lse=None, temperature=1.0, grad_output=1.0):
    """Row losses [N] and the student's gradient [N, V]."""
    x = np.asarray(x, np.float64)
    N, V = x.shape
    q = teacher_weights(values, ids, V, lse, temperature)
    loss, grad = np.zeros(N), np.zeros((N, V))
    for r in range(N):
        live = q[r] > 0
        if not live.any():
            continue
        y = x[r] / temperature
        m = y.max()
        at = np.asarray(ids[r])[live]
        with np.errstate(invalid="ignore", divide="ignore"):
            # not logsumexp(y) - y: m + log d is m where m is large
            e = np.exp(y - m) if m > -np.inf else np.zeros(V)
            terms = np.where(y[at] == -np.inf, np.inf, q[r][live] * ((m - y[at]) + np.log(e.sum())))
            p = e / e.sum() if m > -np.inf else e
        loss[r] = temperature ** 2 * terms.sum()
        g = q[r].sum() * p
        np.subtract.at(g, at, q[r][live])
        grad[r] = grad_output * temperature * g
    return loss, grad


def sample_row(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row; settings as they are held in fp32."""
    row = np.asarray(row, np.float64)
    at = order(row)
    at = at[~np.isnan(row[at]) & (row[at] > -np.inf)]
    if len(at) == 0:
        return -1
    if not temperature > 0:
        return int(at[0])
    top = row[at[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((row[at] - top) / np.float64(temperature))
    if top == np.inf:                    # nothing but the +inf, at any temperature
        w = np.zeros_like(w)
    w = np.where(row[at] == top, 1.0, w).astype(np.longdouble)
    if 0 < top_k < len(row):
        at, w = at[:top_k], w[:top_k]
    n = len(at)
    if top_p < 1:
        before = np.concatenate([[0], np.cumsum(w)[:-1]])
        n = max(1, int((before < np.longdouble(np.float64(top_p)) * w.sum()).sum()))
    at, w = at[:n], w[:n]
    if min_p > 0:
        n = max(1, int((w >= min(np.float64(min_p), 1.0)).sum()))
        at, w = at[:n], w[:n]
    by = np.argsort(at)
    at, c = at[by], np.cumsum(w[by])
    u = np.float64(u) if u > 0 else 0.0
    i = int((c <= u * c[-1]).sum())
    return int(at[min(i, int(np.nonzero(w[by] > 0)[0][-1]))])


def embedding(ids, weight, scale):
    ids, weight = np.asarray(ids).reshape(-1), np.asarray(weight, np.float64)
    ok = (ids >= 0) & (ids < len(weight))
    return np.where(ok[:, None], scale * weight[np.where(ok, ids, 0)], 0.0)


def embedding_grad(dy, ids, V, scale, padding_idx=None):
    dy, ids = np.asarray(dy, np.float64), np.asarray(ids).reshape(-1)
    out = np.zeros((V, dy.shape[-1]))
    ok = (ids >= 0) & (ids < V) & (ids != (-1 if padding_idx is None else padding_idx))
    np.add.at(out, ids[ok], dy.reshape(len(ids), -1)[ok])
    return scale * out


def adjust(x, tokens=None, lengths=None, prompts=None, repetition=1.0, frequency=0.0, presence=0.0, bias_ids=None, bias=None,
           allowed=None):
    """Rows x [N, V] with penalties, biases and mask (mga_adjust_logits), and the sum of the
    magnitudes that went into each value."""
    x = np.asarray(x, np.float64)
    N, V = x.shape
    each = lambda v: np.broadcast_to(np.asarray(v, np.float64), (N,))   # noqa: E731
    rep, freq, pres = each(repetition), each(frequency), each(presence)
    y, mag = x.copy(), np.abs(x)
    for r in range(N):
        if tokens is not None:
            n = len(tokens[r]) if lengths is None else min(max(int(lengths[r]), 0), len(tokens[r]))
            m = 0 if prompts is None else min(max(int(prompts[r]), 0), n)
            seen = {int(t) for t in tokens[r][:n] if 0 <= t < V}
            count = {}
            for t in tokens[r][m:n]:
                if 0 <= t < V:
                    count[int(t)] = count.get(int(t), 0) + 1
            f = rep[r] if rep[r] > 0 else 1.0
            for t in seen:
                y[r, t] = y[r, t] / f if y[r, t] > 0 else y[r, t] * f
                mag[r, t] = abs(y[r, t])
                if t in count:
                    y[r, t] -= freq[r] * count[t] + pres[r]
                    mag[r, t] += abs(freq[r]) * count[t] + abs(pres[r])
        if bias_ids is not None:
            for t, b in zip(np.broadcast_to(bias_ids, (N, np.shape(bias_ids)[-1]))[r],
                            np.broadcast_to(bias, (N, np.shape(bias)[-1]))[r]):
                if 0 <= t < V:
                    y[r, int(t)] += float(b)
                    mag[r, int(t)] += abs(float(b))
        if allowed is not None:
            words = np.broadcast_to(allowed, (N, np.shape(allowed)[-1]))[r].astype(np.int64)
            v = np.arange(V)
            y[r][(words[v // 32] >> (v % 32)) & 1 == 0] = -np.inf
    return y, mag
