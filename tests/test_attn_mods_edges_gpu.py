"""Prompt attention with modified scores in the forms of q and output that its other tests take in part only.

Tolerances as in test_attn_mods_gpu, but for a weight: with a split q 2^-21 for the exponential and the two planes of the
probability, whatever the output's type; with a single plane 2^-11 more."""
import numpy as np
import pytest

import test_attn_mods_gpu as base
import token_step_ref as ref
import vsl_testlib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
FORMS = [(True, 1), (True, 2), (True, 3), (False, 1), (False, 2), (False, 3)]


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


def close(got, qv, K, V, pos0, scale, x2, odt, **kw):
    """Whether each output is within its bound."""
    S, _, hd = qv.shape
    want, err = ref.attention(qv, K, V, float(np.float32(scale)), pos0 + np.arange(S), score_rel=2 * hd * U + 6 * U,
                              prob_rel=2.0 ** -21 + (0 if x2 else 2.0 ** -11), **kw)
    a = np.abs(want)
    last = {1: np.maximum(2.0 ** -11 * a, 2.0 ** -25), 2: 2.0 ** -22 * a + 2.0 ** -25, 3: 2.0 ** -15 * a + 2.0 ** -19}[odt]
    return np.abs(got - want) <= (err + last) * 1.001 + 2 * U * a


@pytest.mark.parametrize("hd,n_q,n_kv", [(64, 8, 1), (128, 6, 2), (128, 32, 8)])
@pytest.mark.parametrize("S,pos0", [(45, 0), (150, 70), (33, 900)])
def test_split_q_keeps_its_digits(vsl, H, dev, hd, n_q, n_kv, S, pos0):
    """A split q has split probabilities, as in attention without modifications: with an fp16 output too its own rounding is all
    that is lost. (Values of one sign per dim would hide it: outputs near 0 are what shows a weight's rounding.)"""
    rng = np.random.default_rng(S + hd)
    K, V, kc, vc = base.caches(rng, n_kv, pos0 + S, hd, pos0 + S + 9, np.float16)
    q = rng.normal(0, 2, (S, n_q, hd)).astype(np.float32)
    for kw in (dict(softcap=50.0), dict(softcap=0.0, slopes=base.slopes_of(n_q)), dict(softcap=30.0, ranges=base.packed(S, pos0, rng))):
        m = base.mods(vsl, dev, **kw)
        got, qv = base.prompt(vsl, H, dev, q, kc, vc, pos0, 0.09, m)
        assert np.all(close(got, qv, K, V, pos0, 0.09, True, 1, **kw)), kw


@pytest.mark.parametrize("x2,odt", FORMS)
@pytest.mark.parametrize("hd,S,pos0", [(128, 5, 2500), (64, 64, 1200), (128, 300, 700)])
def test_split_keys_in_every_form(vsl, H, dev, x2, odt, hd, S, pos0):
    rng = np.random.default_rng(S + odt)
    K, V, kc, vc = base.caches(rng, 2, pos0 + S, hd, pos0 + S, np.float16)
    q = rng.normal(0, 2, (S, 4, hd)).astype(np.float32)
    assert H.vsl_attn_prefill_mods_ws_bytes(S, pos0, 4, 2, hd) > 0
    for rg in (None, base.packed(S, pos0, rng)):
        kw = dict(softcap=30.0, slopes=base.slopes_of(4), ranges=rg)
        m = base.mods(vsl, dev, **kw)
        for ws in (True, False):
            got, qv = base.prompt(vsl, H, dev, q, kc, vc, pos0, 0.09, m, x2, odt, ws)
            assert np.all(close(got, qv, K, V, pos0, 0.09, x2, odt, **kw)), (ws, rg is None)


@pytest.mark.parametrize("x2,odt", FORMS)
@pytest.mark.parametrize("hd,pos0", [(64, 0), (128, 0), (64, 900), (128, 900)])
def test_masked_values_stay_out_in_every_form(vsl, H, dev, x2, odt, hd, pos0):
    """A document with infinities and NaN between two others, one of whose tiles it shares; rows of padding; keys split and not."""
    rng = np.random.default_rng(hd + odt)
    S, n_q, n_kv = 100, 4, 2
    K, V, kc, vc = base.caches(rng, n_kv, pos0 + S, hd, pos0 + S + 70, np.float16, stale=np.inf)
    q = rng.normal(0, 1, (S, n_q, hd)).astype(np.float32)
    rg = np.zeros((S, 2), np.uint32)
    for b, e in ((0, 30), (30, 41), (41, 99)):
        for i in range(b, e):
            rg[i] = (pos0 + b, pos0 + i + 1)
    kw = dict(softcap=30.0, slopes=base.slopes_of(n_q), ranges=rg)
    m = base.mods(vsl, dev, **kw)
    for bad in (np.nan, np.inf):
        k2, v2 = kc.copy(), vc.copy()
        k2[:, pos0 + 32:pos0 + 41, ::3] = bad
        v2[:, pos0 + 33, 7] = bad
        for ws in (True, False):
            got, qv = base.prompt(vsl, H, dev, q, k2, v2, pos0, 0.1, m, x2, odt, ws)
            ok = close(got, qv, K, V, pos0, 0.1, x2, odt, **kw)
            assert np.all(ok[np.r_[0:32, 41:100]]), (bad, ws)
            assert not got[99].any()


@pytest.mark.parametrize("x2", [True, False])
def test_caps_from_small_to_large(vsl, H, dev, x2):
    """Caps on both sides of those whose polynomial has coefficients within fp32's range, scores from far below to far above them."""
    rng = np.random.default_rng(31)
    S, hd = 70, 128
    K, V, kc, vc = base.caches(rng, 2, S, hd, S, np.float16)
    q = rng.normal(0, 30, (S, 4, hd)).astype(np.float32)
    for cap in (0.01, 2.0, 89.0, 92.0, 500.0, 2000.0, 2500.0, 1e5, 1e30):
        for scale in (0.0884, 0.002):
            got, qv = base.prompt(vsl, H, dev, q, kc, vc, 0, scale, base.mods(vsl, dev, cap), x2)
            assert np.all(close(got, qv, K, V, 0, scale, x2, 1, softcap=cap)), (cap, scale)


def test_scale_and_cap_near_the_largest_number(vsl, H, dev):
    """Keys of zeros: every score is 0, whatever the scale and the cap, and rows are means of the values."""
    rng = np.random.default_rng(32)
    S, hd = 40, 64
    K, V, kc, vc = base.caches(rng, 1, S, hd, S, np.float16)
    K[:], kc[:] = 0, 0
    q = rng.normal(0, 1, (S, 2, hd)).astype(np.float32)
    for scale, cap in ((3e38, 3e37), (-3e38, 3e37), (3e38, 2e38), (1e-30, 1e-30), (0.0, 2e38), (2e-20, 1e15)):
        got, qv = base.prompt(vsl, H, dev, q, kc, vc, 0, scale, base.mods(vsl, dev, cap), True, 2)
        assert np.all(close(got, qv, K, V, 0, scale, True, 2, softcap=cap)), (scale, cap)
        row = base.decode(vsl, H, dev, q[-1], kc, vc, S - 1, scale, base.mods(vsl, dev, cap), nsplit=3)
        assert base.decode_ok(row, q[-1], K, V, S - 1, scale, np.float16, cap), (scale, cap)
