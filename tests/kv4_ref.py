"""The 4-bit KV cache (VSL_DT_KV4) and its operators in numpy, 64 bits, from the definitions in include/vsl_hip.h."""
import numpy as np

NAN_STEP = 0x7E00
SHIFT = [4 * (e // 2 + 4 * (e % 2)) for e in range(8)]


def positions(cap):
    return (cap + 127) // 128 * 128


def steps_off(n_kv, cap, hd):
    return (n_kv * positions(cap) * hd // 2 + 255) // 256 * 256


def cache_bytes(n_kv, cap, hd):
    return steps_off(n_kv, cap, hd) + n_kv * positions(cap) * (hd // 32) * 2


def quantize(x):
    """Codes [..., hd] and stored steps [..., hd / 32] of rows x."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        lo, hi = np.minimum(b.min(-1), 0.0), np.maximum(b.max(-1), 0.0)
        bad = ~np.isfinite(b).all(-1) | ~(hi - lo <= 65280.0)
        lo, hi = np.where(bad, 0.0, lo), np.where(bad, 0.0, hi)
        f, e = np.frexp((hi - lo) / 15.0)
        d = np.maximum(np.ldexp(np.ceil(np.ldexp(f, 7)), e - 7), 2.0 ** -14)
        z = np.rint(-lo / d)
        n = np.clip(np.rint(np.where(bad[..., None], 0.0, b) / d[..., None]) + z[..., None], 0, 15)
    assert np.all(d.astype(np.float16).astype(np.float64) == d)
    steps = d.astype(np.float16).view(np.uint16) | z.astype(np.uint16)
    steps = np.where(bad, NAN_STEP, steps).astype(np.uint16)
    n = np.where(bad[..., None], 0, n)
    return n.reshape(x.shape).astype(np.uint32), steps


def values(codes, steps):
    """What codes stand for."""
    d = (steps & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64)
    z = (steps & 15).astype(np.float64)
    n = codes.reshape(*codes.shape[:-1], -1, 32).astype(np.float64)
    return ((n - z[..., None]) * d[..., None]).reshape(codes.shape)


def views(buf, n_kv, cap, hd, is_v):
    """(code words, steps) of a cache's bytes, writable."""
    P, at = positions(cap), steps_off(n_kv, cap, hd)
    w = buf[:n_kv * P * hd // 2].view(np.uint32)
    s = buf[at:at + n_kv * P * (hd // 32) * 2].view(np.uint16)
    if is_v:
        return w.reshape(n_kv, P // 8, hd), s.reshape(n_kv, P // 8, hd // 32, 8)
    return w.reshape(n_kv, P, hd // 8), s.reshape(n_kv, P, hd // 32)


def pack(buf, rows, pos0, n_kv, cap, hd, is_v):
    """Rows [n_kv][n][hd] into a cache's bytes at pos0, the other positions' bits kept."""
    w, s = views(buf, n_kv, cap, hd, is_v)
    codes, steps = quantize(rows)
    for i in range(rows.shape[1]):
        p = pos0 + i
        if is_v:
            sh = SHIFT[p % 8]
            w[:, p // 8] = (w[:, p // 8] & np.uint32(0xFFFFFFFF ^ (15 << sh))) | (codes[:, i] << np.uint32(sh))
            s[:, p // 8, :, p % 8] = steps[:, i]
        else:
            c = codes[:, i].reshape(n_kv, hd // 8, 8)
            w[:, p] = sum(c[..., e] << np.uint32(SHIFT[e]) for e in range(8))
            s[:, p] = steps[:, i]


def unpack(buf, pos0, n, n_kv, cap, hd, is_v):
    """The values of positions pos0 .. pos0 + n - 1, [n_kv][n][hd] in 64 bits."""
    w, s = views(buf, n_kv, cap, hd, is_v)
    sh = np.array(SHIFT, np.uint32)
    p = np.arange(pos0, pos0 + n)
    if is_v:
        codes = (w[:, p // 8] >> sh[p % 8][None, :, None]) & 15
        steps = s[:, p // 8, :, p % 8].transpose(1, 0, 2) if n else s[:, :0, :, 0]
    else:
        codes = ((w[:, p][..., None] >> sh) & 15).reshape(n_kv, n, hd)
        steps = s[:, p]
    with np.errstate(all="ignore"):
        return values(codes, steps)


def append(qkv, n_q, n_kv, hd, pos0, gq, gk, eps, halves, cos, sin):
    """q [S][n_q][hd], k and v [n_kv][S][hd] after norms and rotation, 64 bits."""
    S = qkv.shape[0]
    y = np.asarray(qkv, np.float64).reshape(S, n_q + 2 * n_kv, hd)
    c, s = (t[pos0:pos0 + S, None].astype(np.float64) for t in (cos, sin))

    def rot(x, g):
        if g is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * g.astype(np.float64)
        out = np.empty_like(x)
        a, b = (x[..., :hd // 2], x[..., hd // 2:]) if halves else (x[..., 0::2], x[..., 1::2])
        u, v = a * c - b * s, a * s + b * c
        if halves:
            out[..., :hd // 2], out[..., hd // 2:] = u, v
        else:
            out[..., 0::2], out[..., 1::2] = u, v
        return out

    with np.errstate(all="ignore"):
        return (rot(y[:, :n_q], gq), rot(y[:, n_q:n_q + n_kv], gk).transpose(1, 0, 2),
                y[:, n_q + n_kv:].transpose(1, 0, 2))


def seen(p, n, window):
    """Which of keys 0..n-1 the query at position p attends to; window: None or (window, n_global, threshold)."""
    j = np.arange(n)
    ok = j <= p
    if window is not None and p + 1 > window[2]:
        ok &= (j < window[1]) | (j >= p - window[0])
    return ok


def attend(q, K, V, p0, scale, window=None):
    """Attention of q [S][n_q][hd] at positions p0.. over K, V [n_kv][n][hd]."""
    S, n_q, hd = q.shape
    n_kv, n = K.shape[:2]
    out = np.empty((S, n_q, hd))
    ok = np.stack([seen(p0 + s, n, window) for s in range(S)])
    whole = np.isfinite(K).all() and np.isfinite(V).all()
    with np.errstate(all="ignore"):
        for h in range(n_q):
            k, v = K[h * n_kv // n_q], V[h * n_kv // n_q]
            if whole:
                x = np.where(ok, (q[:, h] @ k.T) * scale, -np.inf)
                w = np.exp(x - x.max(1, keepdims=True))
                out[:, h] = (w @ v) / w.sum(1, keepdims=True)
                continue
            for s in range(S):  # what is not seen takes no part, whatever it holds
                x = (k[ok[s]] @ q[s, h]) * scale
                w = np.exp(x - np.max(x))
                out[s, h] = (w @ v[ok[s]]) / w.sum()
    return out


def tables(cap, hd, theta=10000.0):
    a = np.arange(cap)[:, None] * theta ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
