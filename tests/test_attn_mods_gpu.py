"""Attention with capped scores, a distance bias and key ranges, decode and prompt, against the definition in 64 bits.

Tolerances, from the arithmetic (u = 2^-24; token_step_ref.attention takes them key by key):
  a score   a sum of hd products of fp16 (or fp32) values in 32 bits: hd u of the sum of magnitudes (fp32 caches: the
            products are rounded too, and both factors where they are scaled: 3 u more; decode over fp16 caches and the split
            q: 2^-22 from the planes, and 2^-25 absolute per value, here below 2^-22 of |q| >= 1/8 on average); the factors
            scale, log2 e, 1 / softcap 3 u of the score; tanh 10 u of the capped score; bias 4 u
  a weight  2^-21 for the exponential and the planes of the probability; with a single plane (fp16 q, or
            an fp16 output) 2^-11 more
  sums      over n keys n u of the magnitudes, and 2^-31 for what the planes drop of small probabilities
  outputs   fp16 2^-11 |.| or 2^-25, split 2^-22 |.| + 2^-25, fp16 + fp8 2^-15 |.| + 2^-19"""
import ctypes
import math

import numpy as np
import pytest

import token_step_ref as ref
import vsl_testlib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ALL = 0xFFFFFFFF


@pytest.fixture(scope="module")
def _dev():
    return vsl_testlib.Dev()


@pytest.fixture
def dev(_dev):
    yield _dev
    _dev.release()


@pytest.fixture(scope="module")
def H(vsl):
    return vsl.hip()


def mods(vsl, dev, softcap=0.0, slopes=None, ranges=None):
    s = None if slopes is None else dev.put(np.asarray(slopes, np.float32))
    r = None if ranges is None else dev.put(np.asarray(ranges, np.uint32))
    return vsl.AttnMods(softcap=softcap, slopes=dev.p(s), ranges=dev.p(r))


def slopes_of(n_q):
    return (2.0 ** (-8.0 * np.arange(1, n_q + 1) / n_q)).astype(np.float32)


def caches(rng, n_kv, n, hd, cap, kt, stale=np.nan):
    """K, V rows as stored, in caches that hold `stale` behind them."""
    K, V = (rng.normal(0, 1, (n_kv, n, hd)).astype(kt) for _ in range(2))
    kc, vc = (np.full((n_kv, cap, hd), stale, kt) for _ in range(2))
    kc[:, :n], vc[:, :n] = K, V
    return K.astype(np.float64), V.astype(np.float64), kc, vc


# ------------------------------------------------------------------------------------------
# decode
# ------------------------------------------------------------------------------------------
def decode(vsl, H, dev, q, kc, vc, pos, scale, m, nsplit=32, ctrl=None, out=None):
    n_kv, cap, hd = kc.shape
    n_q = q.shape[0]
    d = [dev.put(a) for a in (q.astype(np.float32), kc, vc)]
    po, pml = dev.put(np.full(n_q * nsplit * hd, np.nan, np.float32)), dev.put(np.full(n_q * nsplit * 2, np.nan, np.float32))
    o = dev.put(np.full((n_q, hd), 55, np.float32))
    c = dev.put(np.array([pos, 0, 0, 0, 9, 0, cap, 0] if ctrl is None else ctrl, np.uint32))
    vsl.check(H.vsl_attn_decode_mods(dev.p(d[0]), dev.p(d[1]), dev.p(d[2]), vsl.VSL_DT_F16 if kc.dtype == np.float16 else 0, n_q,
                                     n_kv, hd, cap, scale, nsplit, dev.p(po), dev.p(pml), dev.p(o), dev.p(c),
                                     None if m is None else ctypes.byref(m), None))
    return dev.get(o).astype(np.float64)


def decode_ok(got, q, K, V, pos, scale, kt, softcap=0.0, slopes=None, ranges=None):
    hd = q.shape[1]
    rel = hd * U + (2.0 ** -21 if kt == np.float16 else 0) + 6 * U
    want, err = ref.attention(q[None].astype(np.float32).astype(np.float64), K, V, float(np.float32(scale)), [pos], softcap, slopes, ranges, rel,
                              2.0 ** -21)
    return np.all(np.abs(got - want[0]) <= err[0] + 2 * U * np.abs(want[0]) + 1e-30)


GEOMS = [(4, 4, 64), (6, 2, 128), (32, 8, 128), (8, 1, 64), (7, 1, 128), (5, 1, 64)]
DECODE = [(0, 0.0, False, None), (1, 30.0, False, None), (31, 0.0, True, None), (32, 50.0, True, None),
          (40, 50.0, False, (7, ALL)), (129, 5.0, True, (100, 120)), (777, 50.0, False, None), (2500, 30.0, True, (33, 2000)),
          (300, 50.0, True, (299, ALL)), (300, 0.0, False, (300, 301))]


@pytest.mark.parametrize("kt", [np.float16, np.float32])
@pytest.mark.parametrize("geom", GEOMS)
def test_decode(vsl, H, dev, geom, kt):
    n_q, n_kv, hd = geom
    rng = np.random.default_rng(hd + n_q)
    for pos, cap, biased, rg in DECODE:
        K, V, kc, vc = caches(rng, n_kv, pos + 1, hd, pos + 5, kt)
        q = rng.normal(0, 2.5, (n_q, hd)).astype(np.float32)
        sl = slopes_of(n_q) if biased else None
        ranges = None if rg is None else [rg]
        scale = 1 / math.sqrt(hd)
        got = decode(vsl, H, dev, q, kc, vc, pos, scale, mods(vsl, dev, cap, sl, ranges), nsplit=[32, 1, 5, 64][pos % 4])
        assert decode_ok(got, q, K, V, pos, scale, kt, cap, sl, ranges), (pos, cap, biased, rg)


@pytest.mark.parametrize("kt", [np.float16, np.float32])
def test_decode_ranges_without_keys(vsl, H, dev, kt):
    """Zeros, whatever the cache holds; a range past the position has no keys either."""
    rng = np.random.default_rng(1)
    _, _, kc, vc = caches(rng, 2, 20, 64, 64, kt)
    q = rng.normal(0, 1, (4, 64)).astype(np.float32)
    for rg in ((5, 5), (9, 3), (20, 30), (0, 0), (ALL, ALL)):
        assert np.all(decode(vsl, H, dev, q, kc, vc, 19, 0.125, mods(vsl, dev, 50.0, None, [rg])) == 0), rg


@pytest.mark.parametrize("kt", [np.float16, np.float32])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_masked_values_stay_out(vsl, H, dev, hd, kt):
    """Infinities and NaN before and behind the range change no bit; in it, they show."""
    rng = np.random.default_rng(2)
    pos, rg = 200, [(37, 150)]
    K, V, kc, vc = caches(rng, 2, pos + 1, hd, 256, kt, stale=0)
    q = rng.normal(0, 1, (6, hd)).astype(np.float32)
    m = mods(vsl, dev, 30.0, slopes_of(6), rg)
    clean = decode(vsl, H, dev, q, kc, vc, pos, 0.1, m, nsplit=3)
    for bad in (np.nan, np.inf, -np.inf):
        k2, v2 = kc.copy(), vc.copy()
        for c in (k2, v2):
            c[:, :37], c[:, 150:] = bad, bad
        assert np.array_equal(decode(vsl, H, dev, q, k2, v2, pos, 0.1, m, nsplit=3), clean)
    v2 = vc.copy()
    v2[1, 60, 5] = np.inf
    got = decode(vsl, H, dev, q, kc, v2, pos, 0.1, m, nsplit=3)
    # (infinity, or NaN: the planes of a weight are its rounding and what that leaves, 0 or below 0 at times)
    assert not np.any(np.isfinite(got[3:, 5])) and np.array_equal(np.delete(got, 5, 1)[3:], np.delete(clean, 5, 1)[3:])
    k2 = kc.copy()
    k2[0, 60, 5] = np.nan
    got = decode(vsl, H, dev, q, k2, vc, pos, 0.1, m, nsplit=3)
    assert np.all(np.isnan(got[:3])) and np.array_equal(got[3:], clean[3:])


@pytest.mark.parametrize("kt", [np.float16, np.float32])
def test_decode_large_scores(vsl, H, dev, kt):
    """Scores far past the cap (tanh is 1 to all digits), without one far apart, and a negative scale."""
    rng = np.random.default_rng(3)
    K, V, kc, vc = caches(rng, 2, 300, 128, 300, kt)
    q = rng.normal(0, 400, (4, 128)).astype(np.float32)
    for scale, cap in ((0.5, 20.0), (-0.01, 30.0), (0.002, 0.0), (-0.002, 3.0)):
        got = decode(vsl, H, dev, q, kc, vc, 299, scale, mods(vsl, dev, cap))
        assert decode_ok(got, q, K, V, 299, scale, kt, cap), (scale, cap)


def test_decode_flat_tail(vsl, H, dev):
    """16000 equal scores far below one: each of their weights is small, their sum is not."""
    n, hd = 16001, 64
    K, V = np.zeros((1, n, hd), np.float16), np.zeros((1, n, hd), np.float16)
    K[0, 0, 0] = 8
    V[0, 1:] = 1
    q = np.zeros((1, hd), np.float32)
    q[0, 0] = 1
    got = decode(vsl, H, dev, q, K, V, n - 1, 1.0, None)
    w = math.exp(8)
    assert np.all(np.abs(got - 16000 / (16000 + w)) <= 16000 / (16000 + w) * (n * 2 * U + 2.0 ** -20))


def test_decode_without_mods_is_plain_attention(vsl, H, dev):
    rng = np.random.default_rng(4)
    K, V, kc, vc = caches(rng, 8, 500, 128, 512, np.float16, stale=0)
    q = rng.normal(0, 1, (32, 128)).astype(np.float32)
    got = decode(vsl, H, dev, q, kc, vc, 499, 0.09, None)
    d = [dev.put(a) for a in (q, kc, vc)]
    po, pml, o = dev.empty((32 * 32 * 128,), np.float32), dev.empty((32 * 32 * 2,), np.float32), dev.empty((32, 128), np.float32)
    c = dev.put(np.array([499, 0, 0, 0, 9, 0, 512, 0], np.uint32))
    vsl.check(H.vsl_attn_decode(dev.p(d[0]), dev.p(d[1]), dev.p(d[2]), 1, 32, 8, 128, 512, 0.09, 32, dev.p(po), dev.p(pml),
                                dev.p(o), dev.p(c), None))
    assert np.allclose(got, dev.get(o), rtol=0, atol=3e-6)


def test_decode_done(vsl, H, dev):
    rng = np.random.default_rng(5)
    _, _, kc, vc = caches(rng, 1, 8, 64, 8, np.float16)
    q = rng.normal(0, 1, (2, 64)).astype(np.float32)
    assert np.all(decode(vsl, H, dev, q, kc, vc, 0, 0.1, None, ctrl=[7, 0, 1, 0, 9, 0, 8, 0]) == 55)


# ------------------------------------------------------------------------------------------
# prompt
# ------------------------------------------------------------------------------------------
def prompt(vsl, H, dev, q, kc, vc, pos0, scale, m, x2=True, odt=1, ws=True):
    S, n_q, hd = q.shape
    n_kv, cap, _ = kc.shape
    hi = q.astype(np.float16)
    planes = np.stack([hi, (q - hi.astype(np.float32)).astype(np.float16)]) if x2 else hi[None]
    qd, kd, vd = dev.put(planes), dev.put(kc), dev.put(vc)
    n = S * n_q * hd
    o = dev.put(np.full(n * 4 + 64, 0x55, np.uint8))
    size = H.vsl_attn_prefill_mods_ws_bytes(S, pos0, n_q, n_kv, hd) if ws else 0
    w = dev.put(np.full(max(size, 16), 0xFF, np.uint8))
    vsl.check(H.vsl_attn_prefill_mods(dev.p(qd), 2 if x2 else 1, dev.p(kd), dev.p(vd), S, pos0, n_q, n_kv, hd, cap, scale, dev.p(o),
                                      odt, None if m is None else ctypes.byref(m), dev.p(w) if ws else None, size, None))
    raw = dev.get(o)
    used = n * {1: 2, 2: 4, 3: 3}[odt]
    assert np.all(raw[used:] == 0x55)
    hi = raw[:2 * n].view(np.float16).astype(np.float64)
    if odt == 2:
        hi = hi + raw[2 * n:4 * n].view(np.float16).astype(np.float64)
    if odt == 3:
        hi = vsl_testlib.f16f8_value(raw[:2 * n].view(np.float16).reshape(S, n_q * hd), raw[2 * n:3 * n].reshape(S, n_q * hd))
    return hi.reshape(S, n_q, hd), planes.astype(np.float64).sum(0)


def prompt_ok(got, qv, K, V, pos0, scale, x2, odt, softcap=0.0, slopes=None, ranges=None):
    S, _, hd = qv.shape
    want, err = ref.attention(qv, K, V, float(np.float32(scale)), pos0 + np.arange(S), softcap, slopes, ranges,
                              2 * hd * U + 6 * U, 2.0 ** -21 if x2 and odt != 1 else 2.0 ** -11 + 2.0 ** -21)
    a = np.abs(want)
    last = {1: np.maximum(2.0 ** -11 * a, 2.0 ** -25), 2: 2.0 ** -22 * a + 2.0 ** -25, 3: 2.0 ** -15 * a + 2.0 ** -19}[odt]
    return np.all(np.abs(got - want) <= (err + last) * 1.001 + 2 * U * a)


def packed(S, pos0, rng):
    """Documents of 1 to 90 rows, the first behind the cache, rows of padding among them, a prefix that sees itself whole."""
    r = np.zeros((S, 2), np.uint32)
    at = 0
    while at < S:
        n = min(int(rng.integers(1, 90)), S - at)
        kind = rng.integers(0, 4)
        first = 0 if at == 0 else pos0 + at
        for i in range(at, at + n):
            if kind == 0 and at:
                r[i] = (7, 7) if i % 2 else (9, 3)
            elif kind == 1:
                r[i] = (first, max(pos0 + i + 1, pos0 + at + n // 2))
            else:
                r[i] = (first, pos0 + i + 1)
        at += n
    return r


PROMPT = [(1, 0, True, 1), (2, 63, False, 2), (31, 0, True, 3), (33, 64, True, 1), (45, 301, False, 1), (130, 17, True, 2),
          (200, 0, True, 1)]


@pytest.mark.parametrize("geom", GEOMS)
@pytest.mark.parametrize("shape", PROMPT)
def test_prompt(vsl, H, dev, geom, shape):
    n_q, n_kv, hd = geom
    S, pos0, x2, odt = shape
    rng = np.random.default_rng(S + hd)
    K, V, kc, vc = caches(rng, n_kv, pos0 + S, hd, pos0 + S + 9, np.float16)
    q = rng.normal(0, 2.5, (S, n_q, hd)).astype(np.float32)
    scale = 1 / math.sqrt(hd)
    for cap, biased, masked, ws in ((50.0, False, False, True), (0.0, True, True, True), (5.0, True, True, False)):
        sl = slopes_of(n_q) if biased else None
        rg = packed(S, pos0, rng) if masked else None
        got, qv = prompt(vsl, H, dev, q, kc, vc, pos0, scale, mods(vsl, dev, cap, sl, rg), x2, odt, ws)
        assert prompt_ok(got, qv, K, V, pos0, scale, x2, odt, cap, sl, rg), (cap, biased, masked, ws)


@pytest.mark.parametrize("S,pos0", [(5, 2500), (64, 1200), (300, 700)])
def test_prompt_split_keys(vsl, H, dev, S, pos0):
    """Calls that split the keys over blocks (few rows behind a long cache), with a workspace and without."""
    rng = np.random.default_rng(S)
    K, V, kc, vc = caches(rng, 2, pos0 + S, 128, pos0 + S, np.float16)
    q = rng.normal(0, 2, (S, 4, 128)).astype(np.float32)
    assert H.vsl_attn_prefill_mods_ws_bytes(S, pos0, 4, 2, 128) > 0
    for rg in (None, packed(S, pos0, rng), np.array([(pos0 // 2, pos0 // 2 + 70)] * S)):
        m = mods(vsl, dev, 30.0, slopes_of(4), rg)
        for ws in (True, False):
            got, qv = prompt(vsl, H, dev, q, kc, vc, pos0, 0.09, m, True, 1, ws)
            assert prompt_ok(got, qv, K, V, pos0, 0.09, True, 1, 30.0, slopes_of(4), rg), (ws, rg is None)


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_split_keys_of_short_ranges(vsl, H, dev, hd):
    """Ranges of fewer tiles than a call has chunks, far into the cache: most blocks have no tiles at all, and a wave that is
    through before the others of its block changes nothing of theirs."""
    rng = np.random.default_rng(77)
    S, pos0, n_q, n_kv = 45, 2900, 8, 2
    K, V, kc, vc = caches(rng, n_kv, pos0 + S, hd, pos0 + S, np.float16)
    q = rng.normal(0, 2, (S, n_q, hd)).astype(np.float32)
    at = rng.integers(2600, 2700, S)
    rg = np.stack([at, at + rng.integers(0, 70, S)], 1).astype(np.uint32)
    rg[32:] = [(2000, 2001)] * (S - 32)
    assert H.vsl_attn_prefill_mods_ws_bytes(S, pos0, n_q, n_kv, hd) >= 8 * 64 * n_q * (hd + 2) * 4
    m = mods(vsl, dev, 0.0, slopes_of(n_q), rg)
    first, qv = prompt(vsl, H, dev, q, kc, vc, pos0, 0.09, m)
    assert prompt_ok(first, qv, K, V, pos0, 0.09, True, 1, 0.0, slopes_of(n_q), rg)
    for _ in range(20):
        assert np.array_equal(prompt(vsl, H, dev, q, kc, vc, pos0, 0.09, m)[0], first)


@pytest.mark.parametrize("hd,n_q,n_kv", [(64, 4, 4), (128, 4, 1), (128, 3, 1)])
@pytest.mark.parametrize("pos0", [0, 900])
def test_prompt_masked_values_stay_out(vsl, H, dev, hd, n_q, n_kv, pos0):
    """Packed documents, one of which holds infinities and NaN: the others' rows are as without them."""
    rng = np.random.default_rng(hd)
    S = 100
    K, V, kc, vc = caches(rng, n_kv, pos0 + S, hd, pos0 + S + 70, np.float16, stale=np.inf)
    q = rng.normal(0, 1, (S, n_q, hd)).astype(np.float32)
    docs = [(0, 30), (30, 41), (41, 100)]
    rg = np.zeros((S, 2), np.uint32)
    for b, e in docs:
        for i in range(b, e):
            rg[i] = (pos0 + b, pos0 + i + 1)
    rg[99] = 0  # padding
    m = mods(vsl, dev, 30.0, slopes_of(n_q), rg)
    kw = dict(softcap=30.0, slopes=slopes_of(n_q), ranges=rg)
    clean, qv = prompt(vsl, H, dev, q, kc, vc, pos0, 0.1, m)
    assert prompt_ok(clean, qv, K, V, pos0, 0.1, True, 1, **kw)
    for bad in (np.nan, np.inf, -np.inf):
        k2, v2 = kc.copy(), vc.copy()
        k2[:, pos0 + 32:pos0 + 41, ::3] = bad
        v2[:, pos0 + 33, 7] = bad
        got, _ = prompt(vsl, H, dev, q, k2, v2, pos0, 0.1, m)
        others = np.r_[0:32, 41:100]
        want, err = ref.attention(qv, K, V, float(np.float32(0.1)), pos0 + np.arange(S), **kw, score_rel=2 * hd * U + 6 * U,
                                  prob_rel=2.0 ** -11 + 2.0 ** -21)
        a = np.abs(want)
        ok = np.abs(got - want) <= (err + np.maximum(2.0 ** -11 * a, 2.0 ** -25)) * 1.001 + 2 * U * a
        assert np.all(ok[others]), bad
        assert not np.any(np.isfinite(got[33:41, :, 7])), bad
    # values alone: infinities reach the rows that see them (as infinity or NaN), and their other dims not at all
    v2 = vc.copy()
    v2[:, pos0 + 50, 3] = np.inf
    v2[:, pos0 + 60, 3] = -np.inf
    got, _ = prompt(vsl, H, dev, q, kc, v2, pos0, 0.1, m)
    assert not np.any(np.isfinite(got[50:99, :, 3])) and np.all(got[99] == 0)
    want, err = ref.attention(qv, K, V, float(np.float32(0.1)), pos0 + np.arange(S), **kw, score_rel=2 * hd * U + 6 * U,
                              prob_rel=2.0 ** -11 + 2.0 ** -21)
    ok = np.abs(got - want) <= (err + np.maximum(2.0 ** -11 * np.abs(want), 2.0 ** -25)) * 1.001 + 2 * U * np.abs(want)
    assert np.all(np.delete(ok, 3, 2))


def test_prompt_later_rows_stay_out(vsl, H, dev):
    """Causal rows before a row whose values are NaN."""
    rng = np.random.default_rng(8)
    S, hd = 70, 128
    K, V, kc, vc = caches(rng, 1, S, hd, S, np.float16)
    q = rng.normal(0, 1, (S, 4, hd)).astype(np.float32)
    vc[0, 40] = np.nan
    got, qv = prompt(vsl, H, dev, q, kc, vc, 0, 0.1, None)
    Vc = V.copy()
    want, err = ref.attention(qv[:40], K[:, :40], Vc[:, :40], float(np.float32(0.1)), np.arange(40), score_rel=2 * hd * U + 6 * U,
                              prob_rel=2.0 ** -11 + 2.0 ** -21)
    assert np.all(np.abs(got[:40] - want) <= (err + np.maximum(2.0 ** -11 * np.abs(want), 2.0 ** -25)) * 1.001)
    assert np.all(np.isnan(got[40:]))


@pytest.mark.parametrize("x2", [True, False])
def test_prompt_large_scores(vsl, H, dev, x2):
    rng = np.random.default_rng(9)
    S, hd = 40, 64
    K, V, kc, vc = caches(rng, 2, S, hd, S, np.float16)
    q = rng.normal(0, 300, (S, 4, hd)).astype(np.float32)
    for scale, cap in ((0.5, 20.0), (-0.01, 30.0), (0.003, 0.0), (-0.003, 0.0)):
        got, qv = prompt(vsl, H, dev, q, kc, vc, 0, scale, mods(vsl, dev, cap), x2)
        assert prompt_ok(got, qv, K, V, 0, scale, x2, 1, cap), (scale, cap)


def test_prompt_without_mods_is_plain_attention(vsl, H, dev):
    rng = np.random.default_rng(10)
    S, pos0 = 150, 70
    K, V, kc, vc = caches(rng, 8, pos0 + S, 128, 256, np.float16, stale=0)
    q = rng.normal(0, 1, (S, 32, 128)).astype(np.float32)
    got, qv = prompt(vsl, H, dev, q, kc, vc, pos0, 0.09, None, True, 2)
    hi = q.astype(np.float16)
    d = [dev.put(a) for a in (np.stack([hi, (q - hi.astype(np.float32)).astype(np.float16)]), kc, vc)]
    o = dev.empty((2, S, 32, 128), np.float16)
    vsl.check(H.vsl_attn_prefill(dev.p(d[0]), 2, dev.p(d[1]), dev.p(d[2]), S, pos0, 32, 8, 128, 256, 0.09, dev.p(o), 2, None))
    assert np.allclose(got, dev.get(o).astype(np.float64).sum(0), rtol=0, atol=3e-6)
