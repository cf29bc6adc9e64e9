"""Plain 64-bit implementations (numpy) of the scored router, the 8-bit integer
products and the token log probabilities, from their definitions."""
from __future__ import annotations

import numpy as np


def route(z, k, score="softmax", bias=None, available=None, groups=1, kept=1, group_top=2, norm=True, scale=1.0):
    """ids (T, k), weights (T, k) of logits z (T, E) in float64."""
    z = np.asarray(z, np.float64)
    T, E = z.shape
    ids = np.full((T, k), -1, np.int64)
    w = np.zeros((T, k))
    for t in range(T):
        on = [e for e in range(E) if z[t, e] > -np.inf and (available is None or available[e])]
        if not on:
            continue
        top = max(z[t, e] for e in on)
        if score == "softmax":
            raw = {e: 1.0 if z[t, e] == top else np.exp(z[t, e] - top) for e in on}
            total = sum(raw.values())
            s = {e: v / total for e, v in raw.items()}
        else:
            with np.errstate(over="ignore"):
                s = {e: 1.0 / (1.0 + np.exp(-z[t, e])) for e in on}
        if bias is None:
            c = dict(s) if groups > 1 else {e: z[t, e] for e in on}
            order_in = {e: z[t, e] for e in on}
        else:
            c = {e: s[e] + float(bias[e]) for e in on if s[e] + float(bias[e]) > -np.inf}
            order_in = c
        allowed = set(c)
        if groups > 1 and kept < groups:
            per = E // groups
            gs = {}
            for g in range(groups):
                vals = sorted((c[e] for e in c if e // per == g), reverse=True)
                if vals:
                    gs[g] = sum(vals[:group_top])
            best = sorted(gs, key=lambda g: (-gs[g], g))[:kept]
            allowed = {e for e in c if e // per in best}
        chosen = sorted(allowed, key=lambda e: (-order_in[e], e))[:k]
        ids[t, :len(chosen)] = chosen
        if not chosen:
            continue
        if norm:
            # ratios of the scores, also where all of them underflow
            zs = np.array([z[t, e] for e in chosen])
            M = zs.max()
            if score == "softmax":
                v = np.where(zs == M, 1.0, np.exp(np.where(zs == M, 0.0, zs - M)))
            elif M < 0:
                v = np.exp(zs - M) / (1 + np.exp(zs))
            else:
                v = 1 / (1 + np.exp(-zs))
            v = v / v.sum()
        else:
            v = np.array([s[e] for e in chosen])
        w[t, :len(chosen)] = v * scale
    return ids, w


def logprobs(z, tokens, n):
    """dict(logprob, rank, entropy, top_ids, top_logprobs) of logits z (T, V)."""
    z = np.asarray(z, np.float64)
    T, V = z.shape
    out = dict(logprob=np.full(T, np.nan), rank=np.full(T, -1), entropy=np.full(T, np.nan),
               top_ids=np.full((T, n), -1), top_logprobs=np.full((T, n), np.nan))
    for t in range(T):
        row, tok = z[t], int(tokens[t])
        ok = 0 <= tok < V
        if np.isnan(row).any():
            continue
        m = row.max()
        out["top_logprobs"][t] = -np.inf
        order = np.lexsort((np.arange(V), -row))
        if ok:
            out["rank"][t] = int((row > row[tok]).sum() + (row[:tok] == row[tok]).sum())
        if m == -np.inf:
            out["entropy"][t] = 0.0
            if ok:
                out["logprob"][t] = -np.inf
            continue
        d = np.where(row == m, 0.0, row - (m if np.isfinite(m) else 0.0))
        e = np.where(row == m, 1.0, np.exp(d) if np.isfinite(m) else 0.0)
        first = int(np.argmax(row))
        rest = np.delete(e, first).sum()
        ls = np.log1p(rest)
        lp = np.where(row == m, -ls, d - ls) if np.isfinite(m) else np.where(row == m, -ls, -np.inf)
        out["entropy"][t] = ls - np.where(e > 0, e * np.where(e > 0, d, 0.0), 0.0).sum() / (1 + rest)
        if ok:
            out["logprob"][t] = lp[tok]
        for j, v in enumerate(order[:n]):
            if row[v] > -np.inf:
                out["top_ids"][t, j] = v
                out["top_logprobs"][t, j] = lp[v]
    return out


def quantise(x):
    """(codes, scales) of rows in float64: the nearest whole numbers to 127 x / max|x|, ties to even."""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(-1, keepdims=True)
    return np.rint(x * 127 / np.where(top > 0, top, 1)), top / 127


def linear(x, codes, scales):
    q, s = quantise(x)
    return (q @ np.asarray(codes, np.float64).T) * s * np.asarray(scales, np.float64)


def experts(x, ids, weights, gate, up, down, residual=None):
    """gate / up / down: (codes (E, rows, cols), scales (E, rows)) pairs."""
    x = np.asarray(x, np.float64)
    out = np.zeros_like(x) if residual is None else np.asarray(residual, np.float64).copy()
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if not 0 <= e < gate[0].shape[0]:
                continue
            g = linear(x[t:t + 1], gate[0][e], gate[1][e])
            u = linear(x[t:t + 1], up[0][e], up[1][e])
            a = g / (1 + np.exp(-g)) * u
            out[t] += float(weights[t, j]) * linear(a, down[0][e], down[1][e])[0]
    return out
