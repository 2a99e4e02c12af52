"""The paged key-value cache, restated in numpy. TEST INFRASTRUCTURE ONLY.

Pools are [P, KV, page, ...]; entry i of sequence b lies in page table[b, i // page] at row
i % page. Attention is computed in float64 from the definition, the choice of what leaves by
sorting, the moves one by one.
"""
from __future__ import annotations

import numpy as np


def entry(table: np.ndarray, page: int, b: int, i) -> tuple:
    """(page id, row) of entry i (or of an array of entries)."""
    i = np.asarray(i)
    return table[b, i // page], i % page


def entries(pages: np.ndarray, table: np.ndarray, b: int, h: int, n: int) -> np.ndarray:
    p, r = entry(table, pages.shape[2], b, np.arange(n))
    return pages[p, h, r]


def append(pools, table, lengths, seen, k, v, counts) -> None:
    """In place on (k_pages, v_pages, mass, pos)."""
    kp, vp, mass, pos = pools
    page, at = kp.shape[2], 0
    for b, c in enumerate(counts):
        for i in range(c):
            e = lengths[b] + i
            if e < table.shape[1] * page:
                p, r = entry(table, page, b, e)
                kp[p, :, r], vp[p, :, r], mass[p, :, r], pos[p, :, r] = k[at], v[at], 0.0, seen[b] + i
            at += 1


def _softmax(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(weights, logsumexp) over the last axis; a row of -inf gives zeros and -inf."""
    top = x.max(-1, keepdims=True, initial=-np.inf)
    e = np.exp(x - np.where(np.isfinite(top), top, 0.0))
    s = e.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        return e / np.where(s == 0, 1.0, s), (np.log(s) + np.where(np.isfinite(top), top, 0.0))[..., 0]


def attend(q, kp, vp, table, lengths, window=None, sinks=0, scale=None):
    """(out [B,H,hd], lse [B,H], weights: list per b of [KV, n]) in float64."""
    b, h, d = q.shape
    kv = kp.shape[1]
    g = h // kv
    scale = d ** -0.5 if scale is None else scale
    out, lse, weights = np.zeros((b, h, d)), np.full((b, h), -np.inf), []
    for i in range(b):
        n = int(lengths[i])
        at = np.arange(n)
        see = np.ones(n, bool) if window is None else (at >= n - window) | (at < sinks)
        w = np.zeros((kv, n))
        for j in range(kv):
            k = entries(kp, table, i, j, n).astype(np.float64)[see]
            v = entries(vp, table, i, j, n).astype(np.float64)[see]
            rows = slice(j * g, (j + 1) * g)
            p, lse[i, rows] = _softmax(q[i, rows].astype(np.float64) @ k.T * scale)
            out[i, rows] = p @ v
            w[j, see] = p.sum(0)
        weights.append(w)
    return out, lse, weights


def observe(q, kp, table, lengths, scale=None):
    """Weights of the last W queries, summed: list per b of [KV, n] in float64."""
    b, w, h, d = q.shape
    kv = kp.shape[1]
    g = h // kv
    scale = d ** -0.5 if scale is None else scale
    out = []
    for i in range(b):
        n = int(lengths[i])
        add = np.zeros((kv, n))
        for j in range(kv):
            k = entries(kp, table, i, j, n).astype(np.float64)
            for t in range(max(0, w - n), w):
                x = q[i, t, j * g:(j + 1) * g].astype(np.float64) @ k[: n - w + t + 1].T * scale
                add[j, : n - w + t + 1] += _softmax(x)[0].sum(0)
        out.append(add)
    return out


def select(mass, pos, table, lengths, seen, budget, recent, sinks):
    """Lists per (b, h) of the moves (src, dst)."""
    page, kv = mass.shape[2], mass.shape[1]
    out = []
    for b in range(len(lengths)):
        n, row = int(lengths[b]), []
        for h in range(kv):
            if n <= budget:
                row.append(([], []))
                continue
            m, p = entries(mass, table, b, h, n), entries(pos, table, b, h, n)
            safe = ((p >= 0) & (p < sinks)) | (p >= int(seen[b]) - recent)
            rank = sorted(range(n), key=lambda i: (not safe[i], not np.isnan(m[i]), 0.0 if np.isnan(m[i]) or safe[i]
                                                   else -float(m[i]), i))
            kept = set(rank[:budget])
            row.append(([i for i in range(budget, n) if i in kept], [i for i in range(budget) if i not in kept]))
        out.append(row)
    return out
