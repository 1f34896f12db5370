"""Attention over the 4-bit KV cache where its kernels hand data from wave to wave, read what no append wrote, or add a
long tail of small probabilities. Definitions: kv4_ref; tolerances: those of test_kv4_gpu, unless a test states its own."""
import math

import numpy as np
import pytest

import kv4_ref
from test_kv4_gpu import H, U, _dev, attn_tol, decode, dev, filled, out_tol, prefill  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


SHARED = [  # hd, n_q, n_kv, S, pos0: blocks that share expanded tiles, three tiles and more (64 keys, or 128)
    (128, 64, 8, 160, 200), (64, 64, 8, 160, 200), (128, 64, 8, 270, 130), (64, 64, 8, 270, 150), (128, 48, 8, 200, 64),
    (64, 48, 8, 200, 150), (128, 40, 8, 225, 100), (64, 56, 8, 170, 200)]


@pytest.mark.parametrize("shape", SHARED, ids=str)
def test_prompt_tiles_are_kept_apart(vsl, dev, H, shape):
    """Waves of one block that take unlike paths through its tiles (heads whose scores rise from tile to tile, so that
    their sums are rescaled in each, beside heads without any; every other head a NaN, which never raises its maximum):
    every run bit for bit the first, and the finite heads right."""
    hd, n_q, n_kv, S, pos0 = shape
    rng = np.random.default_rng(sum(shape))
    n, cap = pos0 + S, pos0 + S + 5
    K, V = rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1.3, (n_kv, n, hd))
    K[:, :, 0] = np.arange(n) // 64 * 4.0
    kb, vb, K, V = filled(rng, K, V, cap)
    q = rng.normal(0, 1, (S, n_q, hd)).astype(np.float32)
    q[:, :, 0] = np.where(np.arange(n_q) % 4 == 0, 16.0, 0.0)
    q[:, 1::2, 1] = np.nan
    scale = 1.0 / math.sqrt(hd)
    dk, dv = dev.put(kb), dev.put(vb)
    first, used = prefill(vsl, dev, H, q, True, dk, dv, n_kv, cap, pos0, 2, scale)
    assert np.all(np.isnan(first[:, 1::2]))
    fin = np.arange(0, n_q, 2)
    ref = np.concatenate([kv4_ref.attend(used[:, [h]], K[[h * n_kv // n_q]], V[[h * n_kv // n_q]], pos0, scale) for h in fin], 1)
    tol = attn_tol(np.nan_to_num(used), K, V, scale) + out_tol(ref, 2)
    assert np.all(np.abs(first[:, fin] - ref) <= tol)
    for _ in range(6):
        assert np.array_equal(prefill(vsl, dev, H, q, True, dk, dv, n_kv, cap, pos0, 2, scale)[0], first, equal_nan=True)


# ------------------------------------------------------------------------------------------
# positions that no append wrote
# ------------------------------------------------------------------------------------------
FILLS = ["random", 0x7BF0, 0x7000, 0x6C50, 0xFBF0, 0x7C00, 0xFFFF, 0x6C4F]  # against all NaN, as filled() leaves them


def refill(rng, buf, kept, n_kv, cap, hd, is_v, fill):
    """The cache's bytes with other codes and steps wherever `kept` (a truth value a position) is False."""
    w, s = kv4_ref.views(buf, n_kv, cap, hd, is_v)
    new = np.zeros_like(buf)
    nw, ns = kv4_ref.views(new, n_kv, cap, hd, is_v)
    nw[:] = rng.integers(0, 1 << 32, nw.shape, dtype=np.uint32)
    ns[:] = rng.integers(0, 1 << 16, ns.shape, dtype=np.uint16) if fill == "random" else fill
    at = np.flatnonzero(kept)
    if is_v:
        for p in at:
            m = np.uint32(15 << kv4_ref.SHIFT[p % 8])
            nw[:, p // 8] = (nw[:, p // 8] & ~m) | (w[:, p // 8] & m)
            ns[:, p // 8, :, p % 8] = s[:, p // 8, :, p % 8]
    else:
        nw[:, at], ns[:, at] = w[:, at], s[:, at]
    return new


STALE = [  # hd, n_q, n_kv, S, pos0, window: a row block's own waves; two heads, four, and as the group divides share tiles
    (128, 32, 8, 45, 0, None), (64, 8, 2, 33, 70, None), (64, 3, 1, 3, 0, None), (128, 64, 8, 160, 201, None),
    (64, 32, 8, 290, 0, None), (128, 64, 8, 270, 131, None), (64, 64, 8, 270, 3, None), (128, 48, 8, 200, 65, None),
    (128, 40, 8, 225, 100, None), (64, 56, 8, 170, 201, None), (128, 8, 2, 40, 300, (50, 16, 100)),
    (64, 6, 2, 70, 333, (33, 3, 64)), (128, 64, 8, 270, 400, (70, 20, 100)), (64, 40, 8, 240, 450, (20, 70, 300))]


@pytest.mark.parametrize("shape", STALE, ids=str)
def test_prompt_over_what_was_left_in_the_cache(vsl, dev, H, shape):
    """What a cache holds past the last key, and where a window hides a position from every row, reaches no output, whatever
    the bits: infinite, negative and other steps that no append stores, too."""
    hd, n_q, n_kv, S, pos0, window = shape
    rng = np.random.default_rng(sum(shape[:5]))
    n, cap = pos0 + S, pos0 + S + 40
    kb, vb, K, V = filled(rng, rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1.3, (n_kv, n, hd)), cap)
    q = rng.normal(0, 1, (S, n_q, hd)).astype(np.float32)
    scale = 1.0 / math.sqrt(hd)
    kept = np.zeros(kv4_ref.positions(cap), bool)
    for s in range(S):
        kept[:n] |= kv4_ref.seen(pos0 + s, n, window)
    want, used = prefill(vsl, dev, H, q, True, dev.put(kb), dev.put(vb), n_kv, cap, pos0, 2, scale, window)
    ref = kv4_ref.attend(used, K, V, pos0, scale, window)
    assert np.all(np.abs(want - ref) <= attn_tol(used, K, V, scale) + out_tol(ref, 2))
    for fill in FILLS:
        dk, dv = (dev.put(refill(rng, b, kept, n_kv, cap, hd, is_v, fill)) for b, is_v in ((kb, False), (vb, True)))
        got, _ = prefill(vsl, dev, H, q, True, dk, dv, n_kv, cap, pos0, 2, scale, window)
        assert np.array_equal(got, want), fill


@pytest.mark.parametrize("hd,n_q,n_kv,n,nsplit,window", [(128, 8, 2, 45, 4, None), (64, 5, 1, 300, 7, None), (128, 32, 8, 778, 32, None),
                                                         (64, 8, 1, 500, 3, (40, 5, 100)), (128, 4, 4, 700, 8, (100, 33, 64))])
def test_decode_over_what_was_left_in_the_cache(vsl, dev, H, hd, n_q, n_kv, n, nsplit, window):
    rng = np.random.default_rng(n + hd)
    cap = n + 40
    kb, vb, _, _ = filled(rng, rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1.3, (n_kv, n, hd)), cap)
    q = rng.normal(0, 1, (n_q, hd)).astype(np.float32)
    kept = np.zeros(kv4_ref.positions(cap), bool)
    kept[:n] = kv4_ref.seen(n - 1, n, window)
    want = decode(vsl, dev, H, q, dev.put(kb), dev.put(vb), n_kv, cap, n - 1, nsplit, window)
    assert np.isfinite(want).all() and want.any()
    for fill in FILLS:
        dk, dv = (dev.put(refill(rng, b, kept, n_kv, cap, hd, is_v, fill)) for b, is_v in ((kb, False), (vb, True)))
        assert np.array_equal(decode(vsl, dev, H, q, dk, dv, n_kv, cap, n - 1, nsplit, window), want), fill


# ------------------------------------------------------------------------------------------
# one key with nearly all the weight, and a long tail
# ------------------------------------------------------------------------------------------
# The tail's keys have a score of 0, G (in powers of two) below that of key 3, whose value is 0, and one value v: exactly
#   out = t w v / (1 + t w),  w = 2^-G,  t tail keys.
# Probabilities are passed to the second product in binary16, as hi / lo pairs or alone, 2^7 times as large as the reference
# maximum's share (at most 2^8 more): half a subnormal step, 2^-25, is 2^-32 of it, t 2^-32 v of the output. Alone they
# are also rounded by 2^-11 of themselves where they are not subnormal. Relative to the output: a score is off by
# G (2^-22 + (hd + 1) U) as in attn_tol, the exponentials by 2^-22, sums over the keys by 2 n U.
TAIL_GAPS = [25.6, 28.0]


def tail(rng, hd, n_kv, n, cap):
    K, V = np.zeros((n_kv, n, hd)), np.ones((n_kv, n, hd))
    K[:, 3, 0], V[:, 3] = 2.0, 0.0
    return filled(rng, K, V, cap)


def tail_check(got, score, v, t, hd, split, extra):
    """got [..., n_q, hd] of rows that see t tail keys (an array over the leading axes)."""
    w = 2.0 ** -score
    t = np.asarray(t, np.float64).reshape(-1, *[1] * (got.ndim - 1))
    ref = t * w * v / (1 + t * w)
    rel = 2 * (math.log(2) * score * (2.0 ** -22 + (hd + 1) * U) + 2.0 ** -22 + (t + 1) * U) + (0 if split else 2.0 ** -11)
    assert np.all(np.abs(got - ref) <= t * 2.0 ** -32 * v + rel * ref + extra(ref))


@pytest.mark.parametrize("gap", TAIL_GAPS)
@pytest.mark.parametrize("hd,n_q,n_kv,n,nsplit", [(128, 4, 1, 16000, 1), (64, 8, 2, 16001, 1), (128, 8, 1, 30000, 4)])
def test_decode_keeps_a_tail(vsl, dev, H, hd, n_q, n_kv, n, nsplit, gap):
    rng = np.random.default_rng(n)
    cap, scale = n + 9, 1.0 / math.sqrt(hd)
    kb, vb, K, V = tail(rng, hd, n_kv, n, cap)
    a = K[0, 3, 0] * scale * math.log2(math.e)
    q = np.zeros((n_q, hd), np.float32)
    q[:, 0] = gap / a
    got = decode(vsl, dev, H, q, dev.put(kb), dev.put(vb), n_kv, cap, n - 1, nsplit)
    tail_check(got[None], float(q[0, 0]) * a, V[0, 0, 0], n - 1, hd, True, lambda r: 0.0)


@pytest.mark.parametrize("gap", TAIL_GAPS)
@pytest.mark.parametrize("x2", [True, False])
@pytest.mark.parametrize("hd,n_q,n_kv,S,n", [(128, 8, 2, 3, 16000), (64, 4, 1, 40, 16000), (128, 64, 8, 130, 8000), (64, 64, 8, 130, 8000),
                                             (128, 64, 8, 270, 8000), (64, 64, 8, 270, 8000), (128, 40, 8, 225, 8000)])
def test_prompt_keeps_a_tail(vsl, dev, H, hd, n_q, n_kv, S, n, x2, gap):
    rng = np.random.default_rng(n + S)
    cap, scale, pos0 = n + 9, 1.0 / math.sqrt(hd), n - S
    kb, vb, K, V = tail(rng, hd, n_kv, n, cap)
    a = K[0, 3, 0] * scale * math.log2(math.e)
    q = np.zeros((S, n_q, hd), np.float32)
    q[:, :, 0] = gap / a
    got, used = prefill(vsl, dev, H, q, x2, dev.put(kb), dev.put(vb), n_kv, cap, pos0, 2, scale)
    tail_check(got, used[0, 0, 0] * a, V[0, 0, 0], pos0 + np.arange(S), hd, x2, lambda r: out_tol(r, 2))


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 18, 2.0 ** 23])
@pytest.mark.parametrize("hd,n_q,n_kv,S", [(128, 8, 2, 40), (128, 64, 8, 140), (64, 64, 8, 270)])
def test_scores_of_any_size_stay_finite(vsl, dev, H, hd, n_q, n_kv, S, size):
    """Scores so large that fp32 holds them to whole powers of two: the outputs are means of the values all the same."""
    rng = np.random.default_rng(S)
    n, cap, scale = S + 300, S + 320, 1.0 / math.sqrt(hd)
    kb, vb, K, V = filled(rng, rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1, (n_kv, n, hd)), cap)
    q = rng.normal(0, 1, (S, n_q, hd)).astype(np.float32)
    big = size / (np.abs(K).max() * hd ** 0.5 * 4)
    dk, dv = dev.put(kb), dev.put(vb)
    for x2 in (True, False):
        got, _ = prefill(vsl, dev, H, q, x2, dk, dv, n_kv, cap, 300, 2, scale * big)
        assert np.abs(got).max() <= 1.01 * np.abs(V).max()
    one = decode(vsl, dev, H, q[0] * np.float32(min(big, 2.0 ** 12)), dk, dv, n_kv, cap, n - 1, 4)
    assert np.abs(one).max() <= 1.01 * np.abs(V).max()
