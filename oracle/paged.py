"""CPU oracle for the paged 8-bit cache (numpy, float64): appending with norm and
rotation, and the attention of new tokens over it.

TEST INFRASTRUCTURE. Only ``tests/`` imports this module, and only as the checker. Each
function follows the definition in include/mtp_glora_amd.h token by token;
tests/test_oracle_paged.py pins them against other formulations.
"""
from __future__ import annotations

import numpy as np

SCALE_MIN, SCALE_MAX = -100, 119


def e4m3_table():
    """The values of the 256 codes."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >> 7, -v, v)


def round_e4m3(x):
    """Nearest e4m3 value (the even one of two as near), at most 448."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        e = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
        step = 2.0 ** (e - 3)
        r = np.rint(x / step) * step
    return np.where(np.isfinite(x), np.clip(r, -448, 448), np.nan)


def scale_of(amax):
    """The least power of two, 2^-100 .. 2^119, of which 448 hold amax."""
    amax = np.asarray(amax, np.float64)
    m, e = np.frexp(amax)   # amax = m 2^e, m in [0.5, 1)
    k = np.where(amax > 0, e - 9 + (m > 0.875), SCALE_MIN)
    return 2.0 ** np.clip(k, SCALE_MIN, SCALE_MAX)


def prepared(x, weight=None, cos=None, sin=None, eps=1e-6):
    """Rows [T, H, D], normalised and rotated."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    if cos is not None:
        half = x.shape[-1] // 2
        turned = np.concatenate([-x[..., half:], x[..., :half]], -1)
        x = x * np.asarray(cos, np.float64)[:, None] + turned * np.asarray(sin, np.float64)[:, None]
    return x


def places(cu, lengths, table, page_size, num_pages, T):
    """(token, sequence, position, page or None, row) of each new token."""
    for b in range(len(lengths)):
        for t in range(int(cu[b]), min(int(cu[b + 1]), T)):
            pos = int(lengths[b]) + t - int(cu[b])
            i = pos // page_size
            page = int(table[b][i]) if i < len(table[b]) else -1
            yield t, b, pos, (page if 0 <= page < num_pages else None), pos % page_size


def attend(q, k, v, cu, lengths, table, page_size, scale):
    """q [T, Hq, D]; k, v [pages, Hkv, page_size, D] in value (scaled); out [T, Hq, D]
    and sum p |v| alongside."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    out, weight = np.zeros_like(q), np.zeros_like(q)
    held = {}   # a sequence's positions that have a page: position, page, row
    for t, b, pos, _, _ in places(cu, lengths, table, page_size, len(k), T):
        if b not in held:
            j = np.arange(len(table[b]) * page_size)
            ids = np.repeat(np.asarray(table[b], np.int64), page_size)
            there = (ids >= 0) & (ids < len(k))
            held[b] = j[there], ids[there], j[there] % page_size
        j, pg, row = held[b]
        n = int(np.searchsorted(j, pos, side="right"))
        if n == 0:
            continue
        for g in range(k.shape[1]):
            heads = slice(g * G, (g + 1) * G)
            with np.errstate(all="ignore"):
                s = q[t, heads] @ k[pg[:n], g, row[:n]].T * scale
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[t, heads] = p @ v[pg[:n], g, row[:n]]
                weight[t, heads] = p @ np.abs(v[pg[:n], g, row[:n]])
    return out, weight
