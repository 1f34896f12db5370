"""The 4-bit KV cache on the GPU, through the C ABI, against the 64-bit definitions of kv4_ref: the append with its
per-head norms and rotation, the read-back, decode and prompt attention, and a run of them as a token loop makes it.

Tolerances, from the arithmetic (u = 2^-24, half a step of fp32 relative to the value; fp16 2^-11):
  codes and steps  none: they are chosen in 64 bits on both sides
  q fp32           the square sum over hd is 4 multiply-adds and 4 or 5 additions of positive terms (9 u), its mean with eps,
                   the root and the reciprocal add 3 roundings, halved before the last two: 7 u; times x and the gain 9 u;
                   a rotation of (a, b) adds 2 u of each product: 11 u (|a| + |b|), taken as 12. q fp16 and k, v in
                   fp16: 2^-11 |.| more, or half a subnormal step 2^-25; split q 2^-22 |q| + 2^-25 more
  decode           With A = max over keys of sum |q_i k_i| scale log2(e): a score is off by at most
                   A (2^-22 + u) from the hi / lo planes of q and A hd u from the sums, so a probability by
                   ln 2 times twice that plus 2^-22 (its planes) plus 2^-22 (the exponential); sums over n keys add
                   at most n u. An output is a mean of V weighted by them: twice the sum of these, times max |V|.
  prompt           as decode with the split q (without: q is exact, the probabilities are rounded to fp16, 2^-11),
                   plus the rounding of the output, 2^-11 |out| for fp16, 2^-22 |out| + 2^-25 for the split,
                   2^-15 |out| + 2^-19 for fp16 + fp8 (a remainder of at most 2^-11 |out| kept to 2^-4, or to half
                   a subnormal fp8 step, 2^-10, scaled by 2^-12 as its values are)."""
import ctypes
import math

import numpy as np
import pytest

import kv4_ref
import vsl_testlib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5


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


def stale(rng, n_kv, cap, hd):
    """A cache's bytes as earlier use may have left them: any codes, every step a NaN."""
    buf = rng.integers(0, 256, kv4_ref.cache_bytes(n_kv, cap, hd), dtype=np.uint8)
    buf[kv4_ref.steps_off(n_kv, cap, hd):].view(np.uint16)[:] = kv4_ref.NAN_STEP
    return buf


def filled(rng, K, V, cap):
    """Caches holding the rows K, V [n_kv][n][hd] at positions 0.., stale behind them; and the values they stand for."""
    n_kv, n, hd = K.shape
    kb, vb = stale(rng, n_kv, cap, hd), stale(rng, n_kv, cap, hd)
    kv4_ref.pack(kb, K, 0, n_kv, cap, hd, False)
    kv4_ref.pack(vb, V, 0, n_kv, cap, hd, True)
    return kb, vb, kv4_ref.unpack(kb, 0, n, n_kv, cap, hd, False), kv4_ref.unpack(vb, 0, n, n_kv, cap, hd, True)


# ------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------
def _close(got, ref, pair, dt):
    """pair: |a| + |b| of the pair that was rotated (0: not rotated, exact but for the output's type)."""
    a = np.abs(ref)
    last = 0.0 if dt == 0 else np.maximum(2.0 ** -11 * a, 2.0 ** -25) if dt == 1 else 2.0 ** -22 * a + 2.0 ** -25
    return np.all(np.abs(got - ref) <= (12 * U * pair + last) * 1.001)


def _pairs(x, halves):
    """|a| + |b| of every value's pair."""
    a = np.abs(x)
    if halves:
        return a + np.roll(a, x.shape[-1] // 2, -1)
    return a + a.reshape(*x.shape[:-1], -1, 2)[..., ::-1].reshape(x.shape)


APPEND = [  # hd, n_q, n_kv, S, pos0, cap
    (128, 32, 8, 45, 13, 4096), (128, 6, 2, 1, 0, 1), (64, 4, 4, 8, 8, 16), (64, 3, 1, 7, 1, 9), (128, 1, 1, 9, 127, 200),
    (64, 8, 1, 130, 121, 251), (128, 5, 5, 3, 4, 1000), (128, 64, 8, 17, 62, 128)]


@pytest.mark.parametrize("halves", [0, 1])
@pytest.mark.parametrize("shape", APPEND, ids=str)
def test_append_rows(vsl, dev, H, shape, halves):
    hd, n_q, n_kv, S, pos0, cap = shape
    rng = np.random.default_rng(hd + n_q * 7 + S * 131 + pos0 + halves)
    qkv = rng.normal(0, 1.3, (S, (n_q + 2 * n_kv) * hd)).astype(np.float32)
    gq, gk = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2))
    cos, sin = kv4_ref.tables(cap, hd)
    dqkv, dgq, dgk, dc, ds = (dev.put(a) for a in (qkv, gq, gk, cos, sin))
    for n, (use_q, use_k, qdt, kvdt) in enumerate([(1, 1, 2, 7), (1, 0, 0, 7), (0, 1, 1, 7), (0, 0, 2, 7), (1, 1, 1, 1),
                                                   (1, 1, 0, 0)]):
        gains = gq if use_q else None, gk if use_k else None
        q, k, v = kv4_ref.append(qkv, n_q, n_kv, hd, pos0, *gains, EPS, halves, cos, sin)
        q0, k0, _ = kv4_ref.append(qkv, n_q, n_kv, hd, pos0, *gains, EPS, halves, np.ones_like(cos), np.zeros_like(sin))
        planes = 2 if qdt == 2 else 1
        dq = dev.empty((planes, S + 1, n_q, hd) if planes == 1 else (2 * S + 1, n_q, hd), np.float32 if qdt == 0 else np.float16)
        dq.fill_(7.0)
        if kvdt == 7:
            kb, vb = (rng.integers(0, 256, kv4_ref.cache_bytes(n_kv, cap, hd), dtype=np.uint8) for _ in range(2))
        else:
            kb, vb = (rng.normal(0, 1, (n_kv, cap, hd)).astype(np.float16 if kvdt == 1 else np.float32) for _ in range(2))
        dk, dv = dev.put(kb), dev.put(vb)
        vsl.check(H.vsl_qk_norm_rope_append(dev.p(dqkv), S, n_q, n_kv, hd, pos0, dev.p(dgq) if use_q else None,
                                            dev.p(dgk) if use_k else None, EPS, halves, dev.p(dc), dev.p(ds), dev.p(dq), qdt,
                                            dev.p(dk), dev.p(dv), kvdt, cap, None))
        got = dev.get(dq).astype(np.float64).reshape(-1)
        m = S * n_q * hd
        assert np.all(got[planes * m:] == 7.0)
        got = got[:m] + (got[m:2 * m] if planes == 2 else 0.0)
        assert _close(got.reshape(S, n_q, hd), q, _pairs(q0, halves), qdt)
        if kvdt == 7:
            kv4_ref.pack(kb, k, pos0, n_kv, cap, hd, False)
            kv4_ref.pack(vb, v, pos0, n_kv, cap, hd, True)
            assert np.array_equal(dev.get(dk), kb) and np.array_equal(dev.get(dv), vb)  # other positions' bits too
        else:
            for d, b, x, pair in ((dk, kb, k, _pairs(k0, halves)), (dv, vb, v, 0.0)):
                g = dev.get(d)
                assert _close(g[:, pos0:pos0 + S].astype(np.float64), x, pair, kvdt)
                g[:, pos0:pos0 + S] = b[:, pos0:pos0 + S]
                assert np.array_equal(g, b)


@pytest.mark.parametrize("halves", [0, 1])
@pytest.mark.parametrize("hd,n_q,n_kv,kvdt", [(128, 8, 2, 7), (64, 3, 1, 7), (64, 4, 4, 1), (128, 1, 1, 0)])
def test_append_decode_is_append(vsl, dev, H, hd, n_q, n_kv, kvdt, halves):
    """Step by step the same bits as one call over the rows; done and a full cache write nothing."""
    rng = np.random.default_rng(hd + n_q + kvdt)
    cap, pos0, S = 29, 5, 24
    qkv = rng.normal(0, 1.3, (S, (n_q + 2 * n_kv) * hd)).astype(np.float32)
    g = rng.normal(1, 0.2, hd).astype(np.float32)
    cos, sin = kv4_ref.tables(cap, hd)
    dqkv, dg, dc, ds = (dev.put(a) for a in (qkv, g, cos, sin))
    start = rng.integers(0, 120, H.vsl_kv_cache_bytes(kvdt, n_kv, cap, hd), dtype=np.uint8)
    ka, va, kb, vb = (dev.put(start) for _ in range(4))
    qa, qb = dev.empty((S, n_q * hd), np.float32), dev.empty((S, n_q * hd), np.float32)
    vsl.check(H.vsl_qk_norm_rope_append(dev.p(dqkv), S, n_q, n_kv, hd, pos0, dev.p(dg), dev.p(dg), EPS, halves, dev.p(dc),
                                        dev.p(ds), dev.p(qa), 0, dev.p(ka), dev.p(va), kvdt, cap, None))
    ctrl = dev.empty((8,), np.int32)

    def step(i, pos):
        vsl.check(H.vsl_qk_norm_rope_append_decode(
            dqkv[i].data_ptr(), n_q, n_kv, hd, dev.p(dg), dev.p(dg), EPS, halves, dev.p(dc), dev.p(ds), qb[i].data_ptr(),
            dev.p(kb), dev.p(vb), kvdt, cap, dev.p(ctrl), None))

    for i in range(S):
        vsl.check(H.vsl_ctrl_reset(dev.p(ctrl), pos0 + i, 4, 0, cap, None))
        step(i, pos0 + i)
    for a, b in ((qa, qb), (ka, kb), (va, vb)):
        assert np.array_equal(dev.get(a), dev.get(b))
    before = dev.get(kb).copy(), dev.get(vb).copy(), dev.get(qb).copy()
    vsl.check(H.vsl_ctrl_reset(dev.p(ctrl), cap, 4, 0, cap, None))   # past the capacity: done and error
    step(0, cap)
    c = dev.get(ctrl)
    assert c[2] == 1 and c[7] == 1
    vsl.check(H.vsl_ctrl_reset(dev.p(ctrl), 3, 4, 0, cap, None))
    ctrl[2] = 1                                                      # done
    step(1, 3)
    for a, b in zip(before, (kb, vb, qb)):
        assert np.array_equal(a, dev.get(b))


def test_append_special_blocks(vsl, dev, H):
    """Zeros, one value, negatives only, values on the codes' borders, steps at both ends of their range, NaN, infinities
    and ranges past 65280; a row of zeros with a norm."""
    hd, n_kv, cap, S = 64, 1, 64, 16
    rng = np.random.default_rng(4)
    x = rng.normal(0, 1, (S, 3 * hd)).astype(np.float32)
    v = x[:, 2 * hd:]
    v[0] = 0
    v[1] = 0
    v[1, 5] = 3.25
    v[2] = -np.abs(v[2])
    v[3, :32] = np.arange(32) - 7.5            # range 31: ties of codes at the chosen step
    v[3, 32:] = (np.arange(32) - 16) * 0.5     # step exactly 2^k
    v[4] = rng.normal(0, 1e-6, hd)
    v[5] = rng.normal(0, 2.0 ** -15, hd)
    v[6, 0], v[6, 1] = 40000.0, -25280.0       # the widest range
    v[7, 0], v[7, 1] = 40000.0, -25281.0       # one past it
    v[8, 3], v[8, 40] = np.nan, np.inf
    v[9, 31], v[9, 32] = -np.inf, 65504.0
    v[10] = 1e-42                              # fp32 subnormals
    v[11] = 3.0e38
    v[12] = np.ldexp(1.0, rng.integers(-20, 10, hd))
    v[13] = -0.0
    x[14, hd:2 * hd] = 0
    x[15, hd + 3] = np.nan
    gk = np.ones(hd, np.float32)
    cos, sin = kv4_ref.tables(cap, hd)
    q, k, vv = kv4_ref.append(x, 1, 1, hd, 3, None, gk, EPS, 0, cos, sin)
    kb, vb = (rng.integers(0, 256, kv4_ref.cache_bytes(n_kv, cap, hd), dtype=np.uint8) for _ in range(2))
    dk, dv, dq = dev.put(kb), dev.put(vb), dev.empty((S, hd), np.float32)
    vsl.check(H.vsl_qk_norm_rope_append(dev.p(dev.put(x)), S, 1, 1, hd, 3, None, dev.p(dev.put(gk)), EPS, 0, dev.p(dev.put(cos)),
                                        dev.p(dev.put(sin)), dev.p(dq), 0, dev.p(dk), dev.p(dv), vsl.VSL_DT_KV4, cap, None))
    kv4_ref.pack(kb, k, 3, 1, cap, hd, False)
    kv4_ref.pack(vb, vv, 3, 1, cap, hd, True)
    assert np.array_equal(dev.get(dk), kb) and np.array_equal(dev.get(dv), vb)
    out = dev.empty((1, S, hd), np.float32)
    vsl.check(H.vsl_kv4_read(None, dev.p(dv), 1, cap, hd, 3, S, None, dev.p(out), 0, None))
    got = dev.get(out)[0]
    assert np.array_equal(np.isnan(got), np.repeat(~np.isfinite(v.reshape(S, 2, 32)).all(-1) |
                                                   (np.float64(v).reshape(S, 2, 32).max(-1).clip(0) -
                                                    np.float64(v).reshape(S, 2, 32).min(-1).clip(None, 0) > 65280), 32, 1))


@pytest.mark.parametrize("hd,n_kv,cap,pos0,n", [(128, 8, 4096, 13, 45), (64, 3, 7, 0, 7), (64, 1, 1, 0, 1), (128, 2, 300, 255, 40),
                                                (64, 2, 520, 7, 1), (128, 1, 40, 16, 8)])
@pytest.mark.parametrize("dt", [0, 1])
def test_read(vsl, dev, H, hd, n_kv, cap, pos0, n, dt):
    rng = np.random.default_rng(hd + n + pos0)
    K, V = (rng.normal(0, 2, (n_kv, n, hd)) for _ in range(2))
    kb, vb = stale(rng, n_kv, cap, hd), stale(rng, n_kv, cap, hd)
    kv4_ref.pack(kb, K, pos0, n_kv, cap, hd, False)
    kv4_ref.pack(vb, V, pos0, n_kv, cap, hd, True)
    dk, dv = dev.put(kb), dev.put(vb)
    t = np.float32 if dt == 0 else np.float16
    for use in ((1, 1), (1, 0), (0, 1)):
        ko, vo = (dev.empty((n_kv * n * hd + 8,), t) for _ in range(2))
        vsl.check(H.vsl_kv4_read(dev.p(dk) if use[0] else None, dev.p(dv) if use[1] else None, n_kv, cap, hd, pos0, n,
                                 dev.p(ko) if use[0] else None, dev.p(vo) if use[1] else None, dt, None))
        for u, o, b, is_v in ((use[0], ko, kb, False), (use[1], vo, vb, True)):
            g = dev.get(o).astype(np.float64)
            assert np.all(g[n_kv * n * hd:] == 0)
            want = kv4_ref.unpack(b, pos0, n, n_kv, cap, hd, is_v) if u else np.zeros((n_kv, n, hd))
            assert np.array_equal(g[:n_kv * n * hd].reshape(want.shape), want)


# ------------------------------------------------------------------------------------------
# decode attention
# ------------------------------------------------------------------------------------------
def attn_tol(q, K, V, scale, split=True):
    """max over keys of the sums above, as the bound of an output's distance (without its rounding)."""
    n_q, hd = q.shape[-2:]
    G = n_q // K.shape[0]
    A = max(float((np.abs(q[..., h, :]) @ np.abs(K[h // G]).T).max()) for h in range(n_q)) * scale * 1.4427
    score = A * ((2.0 ** -22 + U if split else 0) + hd * U)
    prob = 2 * math.log(2) * score + 2.0 ** -22 + (2.0 ** -22 if split else 2.0 ** -11)
    return 2 * (prob + K.shape[1] * U) * float(np.abs(V).max())


def decode(vsl, dev, H, q, dk, dv, n_kv, cap, pos, nsplit, window=None, noalloc=False, stream=None, scale=None):
    n_q, hd = q.shape
    scale = scale or 1.0 / math.sqrt(hd)
    dq, out, ctrl = dev.put(q), dev.empty((n_q, hd), np.float32), dev.empty((8,), np.int32)
    vsl.check(H.vsl_ctrl_reset(dev.p(ctrl), pos, 4, 0, cap, None))
    dev.sync()
    a = (dev.p(dq), dev.p(dk), dev.p(dv), vsl.VSL_DT_KV4, n_q, n_kv, hd, cap, scale, nsplit)
    if noalloc:
        vsl.check(H.vsl_attn_decode_noalloc(*a, dev.p(out), dev.p(ctrl), stream))
    else:
        po, pml = dev.empty((n_q * nsplit * hd,), np.float32), dev.empty((n_q * nsplit * 2,), np.float32)
        a = a + (dev.p(po), dev.p(pml), dev.p(out), dev.p(ctrl))
        vsl.check(H.vsl_attn_decode_window(*a, *window, stream) if window else H.vsl_attn_decode(*a, stream))
    return dev.get(out).astype(np.float64)


DECODE = [  # hd, n_q, n_kv, cap, length, nsplit
    (128, 32, 8, 4096, 778, 32), (64, 32, 8, 4096, 256, 32), (64, 4, 4, 2048, 41, 32), (128, 6, 2, 1000, 1, 1),
    (128, 8, 1, 129, 129, 3), (64, 5, 1, 64, 7, 2), (64, 7, 1, 300, 33, 1), (128, 2, 1, 700, 640, 5), (64, 3, 1, 128, 128, 1),
    (128, 64, 8, 9000, 8999, 64), (64, 8, 1, 5000, 4097, 100), (128, 4, 4, 31, 31, 1024), (128, 5, 1, 260, 255, 7)]


@pytest.mark.parametrize("shape", DECODE, ids=str)
def test_decode(vsl, dev, H, shape):
    hd, n_q, n_kv, cap, n, nsplit = shape
    rng = np.random.default_rng(n + hd + n_q)
    kb, vb, K, V = filled(rng, rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1.3, (n_kv, n, hd)), cap)
    q = rng.normal(0, 1, (n_q, hd)).astype(np.float32)
    scale = 1.0 / math.sqrt(hd)
    ref = kv4_ref.attend(q[None].astype(np.float64), K, V, n - 1, scale)[0]
    dk, dv = dev.put(kb), dev.put(vb)
    got = decode(vsl, dev, H, q, dk, dv, n_kv, cap, n - 1, nsplit)
    assert np.abs(got - ref).max() <= attn_tol(q.astype(np.float64), K, V, scale)
    # roundings of independent signs: the errors of the scores above, once, over all outputs
    assert np.linalg.norm(got - ref) <= 1e-5 * np.linalg.norm(ref)
    if n_q * nsplit <= 4096:
        again = decode(vsl, dev, H, q, dk, dv, n_kv, cap, n - 1, nsplit, noalloc=True)
        assert np.array_equal(got, again)
    # a window over all positions, and a threshold that is not passed, leave the same set
    for w in ((n, 0, 0), (0, 0, n)):
        again = decode(vsl, dev, H, q, dk, dv, n_kv, cap, n - 1, nsplit, window=w)
        assert np.abs(again - ref).max() <= attn_tol(q.astype(np.float64), K, V, scale)


@pytest.mark.parametrize("hd,n_q,n_kv", [(128, 4, 1), (64, 6, 2)])
def test_decode_every_position(vsl, dev, H, hd, n_q, n_kv):
    """A query that only one key answers returns that key's value, for every position of the first tiles and of the last."""
    rng = np.random.default_rng(hd)
    n, cap = 331, 400
    K, V = np.zeros((n_kv, n, hd)), rng.normal(0, 1, (n_kv, n, hd))
    K[:, np.arange(n), np.arange(n) % hd] = np.where(np.arange(n) // hd % 2, -1.0, 1.0) * 2.0 ** (3 * (np.arange(n) // hd // 2) - 3)
    kb, vb, K, V = filled(rng, K, V, cap)
    dk, dv = dev.put(kb), dev.put(vb)
    for p in list(range(0, 70)) + list(range(n - 70, n)):
        q = np.tile(K[0, p] * 4000.0 / np.abs(K[0, p]).max(), (n_q, 1)).astype(np.float32)
        ref = kv4_ref.attend(q[None].astype(np.float64), K, V, n - 1, 1.0)[0]
        got = decode(vsl, dev, H, q, dk, dv, n_kv, cap, n - 1, 2, scale=1.0)
        # one key of the largest size answers (its score is over 400 above the next)
        assert np.abs(got - ref).max() <= 2 * (2.0 ** -20 + n * U) * np.abs(V).max(), p


@pytest.mark.parametrize("hd,n_q,n_kv,cap,n,window,nsplit", [
    (128, 32, 8, 4096, 3000, (512, 16, 100), 32), (64, 4, 4, 2048, 1000, (100, 3, 64), 8), (128, 8, 1, 2000, 1999, (31, 33, 1000), 4),
    (64, 3, 1, 600, 600, (0, 0, 1), 2), (128, 2, 2, 600, 500, (33, 64, 499), 3), (128, 4, 1, 600, 65, (20, 200, 10), 2),
    (64, 8, 1, 1000, 993, (1, 0, 5), 32), (128, 1, 1, 2000, 1500, (700, 700, 8), 7)])
def test_decode_window(vsl, dev, H, hd, n_q, n_kv, cap, n, window, nsplit):
    """The windowed set; NaN keys and values outside it do not reach the output."""
    rng = np.random.default_rng(n + hd)
    K, V = rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1.3, (n_kv, n, hd))
    out = ~kv4_ref.seen(n - 1, n, window)
    K[:, out], V[:, out] = np.nan, np.inf
    kb, vb, K, V = filled(rng, K, V, cap)
    q = rng.normal(0, 1, (n_q, hd)).astype(np.float32)
    scale = 1.0 / math.sqrt(hd)
    ref = kv4_ref.attend(q[None].astype(np.float64), K, V, n - 1, scale, window)[0]
    got = decode(vsl, dev, H, q, dev.put(kb), dev.put(vb), n_kv, cap, n - 1, nsplit, window)
    assert np.all(np.isfinite(ref))
    assert np.abs(got - ref).max() <= attn_tol(q.astype(np.float64), K[:, ~out], V[:, ~out], scale)


def test_decode_nan_and_done(vsl, dev, H):
    """A NaN value shows in its 32 columns, a NaN key in every column, of the heads that read it; done writes nothing;
    large scores and equal scores; another stream."""
    hd, n_q, n_kv, cap, n = 128, 8, 2, 256, 200
    rng = np.random.default_rng(3)
    K, V = rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1, (n_kv, n, hd))
    q = rng.normal(0, 1, (n_q, hd)).astype(np.float32)
    V2, K2 = V.copy(), K.copy()
    V2[1, 77, 40] = np.nan
    K2[0, 150, 3] = np.inf
    kb, vb, _, _ = filled(rng, K, V2, cap)
    got = decode(vsl, dev, H, q, dev.put(kb), dev.put(vb), n_kv, cap, n - 1, 4)
    want = np.zeros((n_q, hd), bool)
    want[4:, 32:64] = True
    assert np.array_equal(np.isnan(got), want)
    kb, vb, _, _ = filled(rng, K2, V, cap)
    for nsplit in (1, 4, 32):
        got = decode(vsl, dev, H, q, dev.put(kb), dev.put(vb), n_kv, cap, n - 1, nsplit)
        assert np.all(np.isnan(got[:4])) and np.all(np.isfinite(got[4:]))
    kb, vb, Kv, Vv = filled(rng, K, V, cap)
    dk, dv = dev.put(kb), dev.put(vb)
    # equal scores: the mean of the values
    got = decode(vsl, dev, H, np.zeros_like(q), dk, dv, n_kv, cap, n - 1, 8)
    ref = np.repeat(Vv.mean(1), 4, 0)
    assert np.abs(got - ref).max() <= 2 * (n * U + 2.0 ** -21) * np.abs(Vv).max()
    # scores of thousands: a few keys, or one, take all the weight
    big = (q * 300).astype(np.float32)
    ref = kv4_ref.attend(big[None].astype(np.float64), Kv, Vv, n - 1, 1 / math.sqrt(hd))[0]
    got = decode(vsl, dev, H, big, dk, dv, n_kv, cap, n - 1, 8)
    assert np.abs(got - ref).max() <= attn_tol(big.astype(np.float64), Kv, Vv, 1 / math.sqrt(hd))
    s = ctypes.c_void_p()
    vsl.check(H.vsl_stream_create(ctypes.byref(s)))
    a = decode(vsl, dev, H, q, dk, dv, n_kv, cap, n - 1, 8, stream=s)
    vsl.check(H.vsl_stream_sync(s))
    vsl.check(H.vsl_stream_destroy(s))
    assert np.array_equal(a, decode(vsl, dev, H, q, dk, dv, n_kv, cap, n - 1, 8))
    ctrl, out = dev.empty((8,), np.int32), dev.empty((n_q, hd), np.float32)
    ctrl[0], ctrl[2] = 100, 1
    po, pml = dev.empty((n_q * 4 * hd,), np.float32), dev.empty((n_q * 4 * 2,), np.float32)
    vsl.check(H.vsl_attn_decode(dev.p(dev.put(q)), dev.p(dk), dev.p(dv), 7, n_q, n_kv, hd, cap, 0.1, 4, dev.p(po), dev.p(pml),
                                dev.p(out), dev.p(ctrl), None))
    assert not dev.get(out).any()


def test_far_heads(vsl, dev, H):
    """A head whose codes begin past 4 GiB: append, read and both attentions there."""
    import torch
    hd, n_kv, n_q, cap, S, pos0 = 128, 9, 9, 9_000_000, 20, 8_999_970
    nb = H.vsl_kv_cache_bytes(7, n_kv, cap, hd)
    assert 8 * kv4_ref.positions(cap) * hd // 2 > 1 << 32
    dk, dv = (torch.zeros(nb, dtype=torch.uint8, device="cuda") for _ in range(2))
    dev._live += [dk, dv]
    rng = np.random.default_rng(1)
    qkv = rng.normal(0, 1.3, (S, 27 * hd)).astype(np.float32)
    cos, sin = (torch.zeros(cap, hd // 2, device="cuda") for _ in range(2))
    dev._live += [cos, sin]
    cos.fill_(0.6)
    sin.fill_(0.8)
    t = np.full((S, hd // 2), 1, np.float32)
    q, k, v = kv4_ref.append(qkv, 9, 9, hd, 0, None, None, EPS, 1, t * np.float32(0.6), t * np.float32(0.8))
    dq = dev.empty((2, S, 9 * hd), np.float16)
    vsl.check(H.vsl_qk_norm_rope_append(dev.p(dev.put(qkv)), S, 9, 9, hd, pos0, None, None, EPS, 1, dev.p(cos), dev.p(sin),
                                        dev.p(dq), 2, dev.p(dk), dev.p(dv), 7, cap, None))
    ko, vo = dev.empty((n_kv, S, hd), np.float32), dev.empty((n_kv, S, hd), np.float32)
    vsl.check(H.vsl_kv4_read(dev.p(dk), dev.p(dv), n_kv, cap, hd, pos0, S, dev.p(ko), dev.p(vo), 0, None))
    Kv, Vv = kv4_ref.values(*kv4_ref.quantize(k)), kv4_ref.values(*kv4_ref.quantize(v))
    assert np.array_equal(dev.get(ko), Kv) and np.array_equal(dev.get(vo), Vv)
    # the last rows through a window of 10 positions
    out = dev.empty((S, 9 * hd), np.float16)
    vsl.check(H.vsl_attn_prefill_kv4_window(dev.p(dq), 2, dev.p(dk), dev.p(dv), S, pos0, 9, 9, hd, cap, 0.1, dev.p(out), 1, 9, 0, 5,
                                            None))
    ref = kv4_ref.attend(q[10:], Kv, Vv, 10, 0.1, (9, 0, 5))
    got = dev.get(out).astype(np.float64).reshape(S, 9, hd)[10:]
    assert np.all(np.abs(got - ref) <= attn_tol(q, Kv, Vv, 0.1) + 2.0 ** -11 * np.abs(ref))
    got = decode(vsl, dev, H, q[-1].astype(np.float32), dk, dv, n_kv, cap, pos0 + S - 1, 8, window=(9, 0, 5), scale=0.1)
    assert np.abs(got - ref[-1]).max() <= attn_tol(q, Kv, Vv, 0.1) + U * np.abs(ref).max()


# ------------------------------------------------------------------------------------------
# prompt attention
# ------------------------------------------------------------------------------------------
def prefill(vsl, dev, H, q, x2, dk, dv, n_kv, cap, pos0, odt, scale, window=None):
    """Outputs as values in 64 bits, and the q that the kernel was given."""
    S, n_q, hd = q.shape
    hi = q.astype(np.float16)
    lo = (q - hi.astype(np.float32)).astype(np.float16)
    dq = dev.put(np.stack([hi, lo]) if x2 else hi)
    size = S * n_q * hd
    out = dev.empty((size * 2 + 64,), np.float16)
    out.fill_(7.0)
    a = (dev.p(dq), 2 if x2 else 1, dev.p(dk), dev.p(dv), S, pos0, n_q, n_kv, hd, cap, scale, dev.p(out), odt)
    vsl.check(H.vsl_attn_prefill_kv4_window(*a, *window, None) if window else H.vsl_attn_prefill_kv4(*a, None))
    o = dev.get(out)
    h = o[:size]
    used = size if odt == 1 else 2 * size if odt == 2 else size + size // 2
    assert np.all(o[used:] == 7.0)
    if odt == 1:
        val = h.astype(np.float64)
    elif odt == 2:
        val = h.astype(np.float64) + o[size:2 * size].astype(np.float64)
    else:
        val = vsl_testlib.f16f8_value(h.reshape(S, -1), o[size:size + size // 2].view(np.uint8).reshape(S, -1)).reshape(-1)
    used_q = hi.astype(np.float64) + (lo.astype(np.float64) if x2 else 0.0)
    return val.reshape(S, n_q, hd), used_q


def out_tol(ref, odt):
    a = np.abs(ref)
    return 2.0 ** -11 * a if odt == 1 else 2.0 ** -22 * a + 2.0 ** -25 if odt == 2 else 2.0 ** -15 * a + 2.0 ** -19


PROMPT = [  # hd, n_q, n_kv, S, pos0, cap
    (128, 32, 8, 45, 0, 4096), (64, 32, 8, 70, 0, 128), (128, 4, 1, 33, 95, 128), (64, 4, 4, 1, 0, 1), (128, 6, 2, 31, 1, 1000),
    (64, 8, 1, 100, 29, 300), (128, 8, 1, 64, 64, 128), (128, 5, 1, 32, 7, 40), (64, 7, 1, 40, 120, 260), (64, 3, 1, 3, 500, 503),
    (128, 2, 1, 129, 0, 129), (64, 2, 2, 65, 63, 200), (64, 6, 1, 20, 200, 400), (128, 1, 1, 5, 251, 256), (128, 7, 1, 9, 60, 100),
    (64, 5, 1, 34, 94, 128), (128, 3, 1, 10, 310, 400), (64, 1, 1, 50, 300, 384),
    # more heads times row blocks than CUs: blocks that share expanded tiles, two heads, four, and as the group divides
    (128, 32, 8, 300, 21, 400), (64, 32, 8, 290, 0, 300), (128, 64, 8, 270, 130, 400), (64, 64, 8, 270, 3, 273),
    (128, 40, 8, 225, 100, 330), (64, 36, 12, 230, 1, 256), (128, 48, 8, 200, 64, 264), (64, 32, 32, 257, 0, 257),
    (128, 32, 16, 280, 40, 320), (64, 56, 8, 170, 200, 384), (128, 32, 32, 260, 3, 300)]


@pytest.mark.parametrize("x2,odt", [(True, 2), (True, 1), (True, 3), (False, 1), (False, 2)])
@pytest.mark.parametrize("shape", PROMPT, ids=str)
def test_prompt(vsl, dev, H, shape, x2, odt):
    hd, n_q, n_kv, S, pos0, cap = shape
    rng = np.random.default_rng(hd + S + pos0 + n_q)
    n = pos0 + S
    kb, vb, K, V = filled(rng, rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1.3, (n_kv, n, hd)), cap)
    q = rng.normal(0, 1, (S, n_q, hd)).astype(np.float32)
    scale = 1.0 / math.sqrt(hd)
    got, used = prefill(vsl, dev, H, q, x2, dev.put(kb), dev.put(vb), n_kv, cap, pos0, odt, scale)
    ref = kv4_ref.attend(used, K, V, pos0, scale)
    assert np.all(np.abs(got - ref) <= attn_tol(used, K, V, scale, x2) + out_tol(ref, odt))


@pytest.mark.parametrize("hd,n_q,n_kv,S,pos0,cap,window", [
    (128, 4, 1, 100, 300, 512, (50, 16, 100)), (64, 4, 2, 70, 129, 256, (10, 3, 150)), (128, 2, 2, 40, 500, 640, (0, 0, 1)),
    (64, 8, 1, 33, 400, 512, (200, 130, 64)), (128, 3, 1, 64, 0, 128, (8, 1, 30)), (64, 1, 1, 96, 190, 300, (33, 70, 200)),
    (128, 32, 8, 300, 200, 512, (150, 20, 260)), (64, 64, 8, 280, 111, 400, (70, 130, 120)), (128, 64, 8, 270, 0, 300, (40, 3, 100)),
    (64, 40, 8, 240, 250, 500, (0, 65, 300))])
def test_prompt_window(vsl, dev, H, hd, n_q, n_kv, S, pos0, cap, window):
    rng = np.random.default_rng(hd + S + pos0)
    n = pos0 + S
    kb, vb, K, V = filled(rng, rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1.3, (n_kv, n, hd)), cap)
    q = rng.normal(0, 1, (S, n_q, hd)).astype(np.float32)
    scale = 1.0 / math.sqrt(hd)
    got, used = prefill(vsl, dev, H, q, True, dev.put(kb), dev.put(vb), n_kv, cap, pos0, 2, scale, window)
    ref = kv4_ref.attend(used, K, V, pos0, scale, window)
    assert np.all(np.abs(got - ref) <= attn_tol(used, K, V, scale) + out_tol(ref, 2))


@pytest.mark.parametrize("window", [None, (20, 4, 30)])
@pytest.mark.parametrize("hd,n_q,n_kv", [(128, 4, 1), (64, 3, 1), (64, 8, 1), (128, 96, 24), (64, 176, 22), (128, 180, 36)])
def test_prompt_nan_rows(vsl, dev, H, hd, n_q, n_kv, window):
    """NaN keys and values reach exactly the rows (and, for values, the 32 columns) that see them."""
    rng = np.random.default_rng(hd + n_q)
    S, pos0, cap = 90, 37, 256
    n = pos0 + S
    for bad_k, bad_v in (([], [(60, 1)]), ([70], []), ([100], [(2, 0), (101, 1)]), ([], [(126, 0)])):
        K, V = rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1, (n_kv, n, hd))
        K[0, bad_k, 5] = np.nan
        for p, b in bad_v:
            V[0, p, 32 * b + 9] = -np.inf
        kb, vb, Kv, Vv = filled(rng, K, V, cap)
        q = rng.normal(0, 1, (S, n_q, hd)).astype(np.float32)
        got, used = prefill(vsl, dev, H, q, True, dev.put(kb), dev.put(vb), n_kv, cap, pos0, 2, 0.1, window)
        want = np.zeros((S, n_q, hd), bool)
        for s in range(S):
            see = kv4_ref.seen(pos0 + s, n, window)
            G = n_q // n_kv  # the heads that read KV head 0
            want[s, :G] |= bool(see[bad_k].any())
            for p, b in bad_v:
                want[s, :G, 32 * b:32 * b + 32] |= bool(see[p])
        assert np.array_equal(np.isnan(got), want)
        ref = kv4_ref.attend(used, np.nan_to_num(Kv), np.nan_to_num(Vv), pos0, 0.1, window)
        tol = attn_tol(used, np.nan_to_num(Kv), np.nan_to_num(Vv), 0.1) + out_tol(ref, 2)
        assert np.all(np.abs(got - ref)[~want] <= tol[~want])


# ------------------------------------------------------------------------------------------
# the projection, and a run of them all
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("wdt", [0, 1, 4, 5, 6])
def test_norm_gemv(vsl, dev, H, wdt):
    N, K = 771, 1024
    rng = np.random.default_rng(wdt)
    x, g = rng.normal(0, 2, K).astype(np.float32), rng.normal(1, 0.2, K).astype(np.float32)
    w = rng.normal(0, 0.02, (N, K)).astype(np.float32)
    if wdt <= 1:
        w = w.astype(np.float32 if wdt == 0 else np.float16)
        dw, W = dev.put(w), w.astype(np.float64)
    else:
        dw = dev.empty((H.vsl_quant_pack_bytes(wdt, N, K) + 256,), np.uint8)
        off = -dw.data_ptr() % 256
        dw = dw[off:]
        vsl.check(H.vsl_quantize_pack(dev.p(dev.put(w)), 0, N, K, wdt, dev.p(dw), None))
        back = dev.empty((N, K), np.float32)
        vsl.check(H.vsl_dequant_pack(dev.p(dw), wdt, N, K, dev.p(back), 0, None))
        W = dev.get(back).astype(np.float64)
    ctrl = dev.empty((8,), np.int32)
    for gamma in (g, None):
        xn = x.astype(np.float64)
        if gamma is not None:
            xn = xn / np.sqrt((xn * xn).mean() + np.float64(np.float32(EPS))) * g
        y = dev.empty((N + 8,), np.float32)
        vsl.check(H.vsl_norm_gemv(dev.p(dev.put(x)), None if gamma is None else dev.p(dev.put(g)), EPS, dev.p(dw), wdt, N, K,
                                  dev.p(y), dev.p(ctrl) if gamma is None else None, None))
        got = dev.get(y)
        # sums of K products in fp32 (a wave's 64 lanes, 16 products each, then 6 levels; block packs scale each
        # 32-value sum once more) of an x rounded five times
        tol = (np.abs(W) @ np.abs(xn)) * (16 + 6 + 5 + 8) * U * 4
        assert np.all(np.abs(got[:N] - W @ xn) <= tol) and not got[N:].any()
    ctrl[2] = 1
    y = dev.empty((N,), np.float32)
    vsl.check(H.vsl_norm_gemv(dev.p(dev.put(x)), None, EPS, dev.p(dw), wdt, N, K, dev.p(y), dev.p(ctrl), None))
    assert not dev.get(y).any()


@pytest.mark.parametrize("hd,n_q,n_kv,halves,window", [(64, 4, 2, 0, None), (128, 8, 1, 1, None), (128, 2, 2, 0, (16, 4, 40))])
def test_token_loop(vsl, dev, H, hd, n_q, n_kv, halves, window):
    """A prompt in two chunks, then decode steps replayed from one captured graph with other work between them: every
    output against the definitions, the cache against its bytes."""
    import torch
    rng = np.random.default_rng(hd + n_q + halves)
    cap, width, scale = 200, (n_q + 2 * n_kv) * hd, 1.0 / math.sqrt(hd)
    gq, gk = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2))
    cos, sin = kv4_ref.tables(cap, hd)
    dgq, dgk, dc, ds = (dev.put(a) for a in (gq, gk, cos, sin))
    kb, vb = stale(rng, n_kv, cap, hd), stale(rng, n_kv, cap, hd)
    dk, dv = dev.put(kb), dev.put(vb)

    def check(q, got, pos0, odt):
        n = pos0 + q.shape[0]
        K, V = (kv4_ref.unpack(b, 0, n, n_kv, cap, hd, b is vb) for b in (kb, vb))
        ref = kv4_ref.attend(q, K, V, pos0, scale, window)
        tol = attn_tol(q, K, V, scale) * 2 + (out_tol(ref, odt) if odt else 0.0)  # q itself is off by up to 24 u (less than hd u)
        assert np.all(np.abs(got - ref) <= tol)

    pos = 0
    for S in (37, 61):
        qkv = rng.normal(0, 1.3, (S, width)).astype(np.float32)
        dq, out = dev.empty((2, S, n_q * hd), np.float16), dev.empty((2, S, n_q * hd), np.float16)
        vsl.check(H.vsl_qk_norm_rope_append(dev.p(dev.put(qkv)), S, n_q, n_kv, hd, pos, dev.p(dgq), dev.p(dgk), EPS, halves,
                                            dev.p(dc), dev.p(ds), dev.p(dq), 2, dev.p(dk), dev.p(dv), 7, cap, None))
        a = (dev.p(dq), 2, dev.p(dk), dev.p(dv), S, pos, n_q, n_kv, hd, cap, scale, dev.p(out), 2)
        vsl.check(H.vsl_attn_prefill_kv4_window(*a, *window, None) if window else H.vsl_attn_prefill_kv4(*a, None))
        q, k, v = kv4_ref.append(qkv, n_q, n_kv, hd, pos, gq, gk, EPS, halves, cos, sin)
        kv4_ref.pack(kb, k, pos, n_kv, cap, hd, False)
        kv4_ref.pack(vb, v, pos, n_kv, cap, hd, True)
        assert np.array_equal(dev.get(dk), kb) and np.array_equal(dev.get(dv), vb)
        check(q, dev.get(out).astype(np.float64).sum(0).reshape(S, n_q, hd), pos, 2)
        pos += S
    row, q_dev, attn = (dev.empty((w,), np.float32) for w in (width, n_q * hd, n_q * hd))
    ctrl, po, pml = dev.empty((8,), np.int32), dev.empty((n_q * 8 * hd,), np.float32), dev.empty((n_q * 8 * 2,), np.float32)
    s, g = ctypes.c_void_p(), ctypes.c_void_p()
    dev.sync()
    vsl.check(H.vsl_stream_create(ctypes.byref(s)))
    vsl.check(H.vsl_graph_begin(s))
    vsl.check(H.vsl_qk_norm_rope_append_decode(dev.p(row), n_q, n_kv, hd, dev.p(dgq), dev.p(dgk), EPS, halves, dev.p(dc),
                                               dev.p(ds), dev.p(q_dev), dev.p(dk), dev.p(dv), 7, cap, dev.p(ctrl), s))
    a = (dev.p(q_dev), dev.p(dk), dev.p(dv), 7, n_q, n_kv, hd, cap, scale, 8, dev.p(po), dev.p(pml), dev.p(attn), dev.p(ctrl))
    vsl.check(H.vsl_attn_decode_window(*a, *window, s) if window else H.vsl_attn_decode(*a, s))
    vsl.check(H.vsl_graph_end(s, ctypes.byref(g)))
    for step in range(20):
        qkv = rng.normal(0, 1.3, (1, width)).astype(np.float32)
        row.copy_(torch.from_numpy(qkv[0]))
        vsl.check(H.vsl_ctrl_reset(dev.p(ctrl), pos, 100, 0, cap, None))
        torch.ones(1000, device="cuda").sum().item()   # the program's own work between replays
        vsl.check(H.vsl_graph_launch(g, s))
        vsl.check(H.vsl_stream_sync(s))
        q, k, v = kv4_ref.append(qkv, n_q, n_kv, hd, pos, gq, gk, EPS, halves, cos, sin)
        kv4_ref.pack(kb, k, pos, n_kv, cap, hd, False)
        kv4_ref.pack(vb, v, pos, n_kv, cap, hd, True)
        check(q, dev.get(attn).astype(np.float64).reshape(1, n_q, hd), pos, 0)
        pos += 1
    assert np.array_equal(dev.get(dk), kb) and np.array_equal(dev.get(dv), vb)
    vsl.check(H.vsl_graph_destroy(g))
    vsl.check(H.vsl_stream_destroy(s))


def test_two_calls_at_once(vsl, dev, H):
    """Prompt attention (both kernels) and decode attention over the same caches on three streams without a wait between,
    a few times over, and a captured prompt call replayed beside eager ones: bit for bit what each gives alone."""
    hd, n_q, n_kv, cap, n = 128, 32, 8, 900, 800
    rng = np.random.default_rng(91)
    kb, vb, _, _ = filled(rng, rng.normal(0, 1, (n_kv, n, hd)), rng.normal(0, 1, (n_kv, n, hd)), cap)
    dk, dv = dev.put(kb), dev.put(vb)
    streams = [ctypes.c_void_p() for _ in range(3)]
    for s in streams:
        vsl.check(H.vsl_stream_create(ctypes.byref(s)))
    few, many, nsplit = 40, 300, 16
    dq = {S: dev.put(rng.normal(0, 1, (2, S, n_q * hd)).astype(np.float16)) for S in (few, many)}
    q1 = dev.put(rng.normal(0, 1, n_q * hd).astype(np.float32))
    ctrl = dev.empty((8,), np.int32)
    vsl.check(H.vsl_ctrl_reset(dev.p(ctrl), n - 1, 4, 0, cap, None))
    po, pml = dev.empty((n_q * nsplit * hd,), np.float32), dev.empty((n_q * nsplit * 2,), np.float32)

    def prompt(S, out, s):
        vsl.check(H.vsl_attn_prefill_kv4(dev.p(dq[S]), 2, dev.p(dk), dev.p(dv), S, n - S, n_q, n_kv, hd, cap, 0.1, dev.p(out), 2, s))

    def token(out, s):
        vsl.check(H.vsl_attn_decode(dev.p(q1), dev.p(dk), dev.p(dv), 7, n_q, n_kv, hd, cap, 0.1, nsplit, dev.p(po), dev.p(pml),
                                    dev.p(out), dev.p(ctrl), s))

    outs = lambda: [dev.empty((2, few, n_q * hd), np.float16), dev.empty((2, many, n_q * hd), np.float16),
                    dev.empty((n_q * hd,), np.float32)]
    alone = outs()
    dev.sync()
    prompt(few, alone[0], None)
    prompt(many, alone[1], None)
    token(alone[2], None)
    alone = [dev.get(o) for o in alone]
    assert all(np.isfinite(a).all() and a.any() for a in alone)
    graph_out, g = dev.empty((2, many, n_q * hd), np.float16), ctypes.c_void_p()
    vsl.check(H.vsl_graph_begin(streams[0]))
    prompt(many, graph_out, streams[0])
    vsl.check(H.vsl_graph_end(streams[0], ctypes.byref(g)))
    for _ in range(4):
        got = outs()
        graph_out.fill_(0)
        dev.sync()
        vsl.check(H.vsl_graph_launch(g, streams[0]))
        prompt(few, got[0], streams[0])
        prompt(many, got[1], streams[1])
        token(got[2], streams[2])
        for s in streams:
            vsl.check(H.vsl_stream_sync(s))
        assert all(np.array_equal(dev.get(o), a) for o, a in zip(got, alone))
        assert np.array_equal(dev.get(graph_out), alone[1])
    vsl.check(H.vsl_graph_destroy(g))
    for s in streams:
        vsl.check(H.vsl_stream_destroy(s))
