"""64-bit definitions of scaled and partial rotation, attention with modified scores and key ranges, and sampling by
temperature, top-k, top-p and min-p, in numpy."""
import math

import numpy as np


def rope_freqs(rot, theta, scaling=0, factor=1.0, orig=0.0, low=0.0, high=0.0, ff=None):
    j = np.arange(rot // 2, dtype=np.float64)
    f = float(theta) ** (-2.0 * j / rot)
    if ff is not None:
        f = f / np.asarray(ff, np.float64)
    if scaling == 1:
        return f / factor
    if scaling == 2:
        a = np.clip((orig * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return a * f + (1 - a) * f / factor
    if scaling == 3:
        def pair(turns):
            return rot * math.log(orig / (2 * math.pi * turns)) / (2 * math.log(theta))
        lo, hi = (min(max(x, 0.0), rot - 1.0) for x in (math.floor(pair(high)), math.ceil(pair(low))))
        b = np.clip((j - lo) / max(hi - lo, 0.001), 0, 1)
        return (1 - b) * f + b * f / factor
    return f


def rotate(x, cos, sin, rot, halves):
    """x [..., hd] by cos, sin [..., rot/2] (broadcast); and |a| + |b| of each value's pair (0: not rotated)."""
    x = np.asarray(x, np.float64)
    y, pair = x.copy(), np.zeros_like(x)
    i = np.arange(rot // 2)
    one, two = (i, i + rot // 2) if halves else (2 * i, 2 * i + 1)
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * cos - b * sin, a * sin + b * cos
    pair[..., one] = pair[..., two] = np.abs(a) + np.abs(b)
    return y, pair


def attention(q, K, V, scale, pos, softcap=0.0, slopes=None, ranges=None, score_rel=0.0, prob_rel=0.0):
    """Rows q [S][n_q][hd] at positions pos [S] over K, V [n_kv][n][hd] (64-bit values); ranges [S][2] or None.
    Returns out [S][n_q][hd] and a bound of its error where a score's sum of products is off by at most score_rel of the
    sum of their magnitudes and a weight, besides, by prob_rel of itself (see the tests' arithmetic)."""
    S, n_q, hd = q.shape
    n_kv, n, _ = K.shape
    out, err = np.zeros((S, n_q, hd)), np.zeros((S, n_q, hd))
    k = np.arange(n)
    U = 2.0 ** -24
    for h in range(n_q):
        Kh, Vh = K[h * n_kv // n_q], V[h * n_kv // n_q]
        for s in range(S):
            b, e = (0, pos[s] + 1) if ranges is None else (int(ranges[s][0]), min(int(ranges[s][1]), n))
            if b >= e:
                continue
            kk = Kh[b:e]
            sc = scale * (kk @ q[s, h])
            size = abs(scale) * (np.abs(kk) @ np.abs(q[s, h]))
            if softcap:
                d = score_rel * size
                sc = softcap * np.tanh(sc / softcap)
                d = d + 10 * U * np.abs(sc)
            else:
                d = (score_rel + 2 * U) * size
            if slopes is not None:
                bias = float(slopes[h]) * np.abs(pos[s] - k[b:e])
                sc = sc - bias
                d = d + 4 * U * (bias + np.abs(sc))
            p = np.exp(sc - sc.max())
            p /= p.sum()
            rel = np.expm1(d) + prob_rel + 2 * U * np.abs(sc - sc.max())  # the exponent's difference is rounded
            out[s, h] = p @ Vh[b:e]
            err[s, h] = (p * rel) @ np.abs(Vh[b:e]) + np.abs(out[s, h]) * (p @ rel) + 2 * (e - b) * (U + 2.0 ** -31) * (p @ np.abs(Vh[b:e]))
    return out, err


def sample(logits, temperature, top_k, top_p, min_p, u):
    """(token, share of the kept weights, distance of u to the nearest border) of one row of float64 logits."""
    l = np.where(np.isnan(logits), -np.inf, np.minimum(logits, np.finfo(np.float32).max))
    V = l.size
    if np.all(l == -np.inf):
        return 0, 0.0, 1.0
    order = np.lexsort((np.arange(V), -l))
    if not temperature > 0:
        return int(order[0]), 1.0, 1.0
    u = min(max(u, 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    k = V if top_k == 0 else min(top_k, V)
    order = order[:k]
    w = np.exp((l[order] - l[order[0]]) / temperature)
    near = 1.0
    if top_p < 1:
        c = np.cumsum(w)
        cut = max(top_p, 0.0) * c[-1]
        n = 1 + int(np.searchsorted(c, cut))
        if 0 < top_p:
            near = min(near, float(np.min(np.abs(c - cut)) / c[-1]))
        order, w = order[:n], w[:n]
    keep = w >= (min_p if min_p > 0 else 0.0)
    keep[0] = True
    kept = np.sort(order[keep])
    w = np.exp((l[kept] - l.max()) / temperature)
    c = np.cumsum(w)
    i = int(np.searchsorted(c, u * c[-1], side="right"))
    near = min(near, float(np.min(np.abs(c[:-1] - u * c[-1])) / c[-1])) if len(c) > 1 else near
    return int(kept[i]), float(w[i] / c[-1]), near
