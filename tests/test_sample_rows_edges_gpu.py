"""Sampling of rows where weights are far apart: kept tokens of very small weight, and rows whose small weights add up.

Tolerances: tokens are equal, u lying further than 1e-10 from every border, or being 0 (or so small that the first kept token has
it); a share is one fp32 rounding (2^-24) off, and 1e-10 of itself for the sums."""
import numpy as np
import pytest

import test_sample_rows_gpu as base
import token_step_ref as ref
import vsl_testlib

pytestmark = pytest.mark.gpu


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


def row(V, *values, rest=-np.inf):
    l = np.full(V, rest, np.float32)
    for at, x in values:
        l[at] = x
    return l


def lists(n, *starts):
    return np.concatenate([np.arange(s, s + n) for s in starts])


# name: (logits, (temperature, top_k, top_p, min_p), first kept token). Weights of that token, relative to the largest's: e^-31 to
# e^-42 (2^-44.7 to 2^-60.6).
FIRST = {
    "few of a list": (row(2, (0, 0), (1, 40)), (1.0, 2, 1.0, 0.0), 0),
    "list of two slices": (row(5000, (3, 0), (4000, 39)), (1.0, 40, 1.0, 0.0), 3),
    "list with ties": (row(5000, (lists(200, 0, 2048, 4096), 0), (4990, 40)), (1.0, 40, 1.0, 0.0), 0),
    "top-k over the whole row": (row(30000, (29999, 40), rest=0), (1.0, 40, 1.0, 0.0), 0),
    "a slice's sum": (row(5000, (0, 0), (3000, 31)), (1.0, 0, 1.0, 0.0), 0),
    "a slice's sum, min-p": (row(5000, (0, -20), (5, 0), (3000, 40)), (1.0, 0, 1.0, 1e-20), 5),
    "a bin kept whole": (row(5000, (0, 0), (slice(2048, 2348), -5), (3000, 36)), (1.0, 150, 1.0, 0.0), 0),
    "the bin of the cut": (row(5000, (slice(0, 300), -1.5), (4000, 40.5)), (1.0, 250, 1.0, 0.0), 0),
    "the whole row": (row(5000, (0, 19965), (slice(2048, 2348), 19963), (3000, 20000)), (1.0, 150, 1.0, 0.0), 0),
}


@pytest.mark.parametrize("name", FIRST)
def test_first_kept_token(vsl, H, dev, name):
    """u of 0 (and what counts as 0) and one below its share give the first kept token, however small its weight."""
    logits, params, first = FIRST[name]
    us = [0.0, np.nan, -1.0, 1e-30]
    tok, share = base.run(vsl, H, dev, np.tile(logits, (4, 1)), [params] * 4, us)
    t, k, p, m = (float(np.float32(x)) for x in params)
    want, ws, _ = ref.sample(logits.astype(np.float64), t, int(k), p, m, 0.0)
    assert want == first and 2.0 ** -62 < ws < 2.0 ** -44
    assert list(tok) == [first] * 4
    assert np.all(np.abs(share.astype(np.float64) - ws) <= (2.0 ** -24 * 1.001 + 1e-10) * ws)


def test_sum_of_small_weights_over_the_whole_row(vsl, H, dev):
    """2^20 tokens of 0.6 2^-42 of the largest, whose share is 2.4 2^-24 together, where l / T is too large for bins."""
    V = 1 << 20
    logits = np.full(V, 20000 + np.log(0.6) - 42 * np.log(2), np.float32)
    logits[0] = 20000
    params = [(1.0, V - 1, 1.0, 0.0), (1.0, V - 300, 1.0, 0.0)]
    base.check(vsl, H, dev, np.tile(logits, (2, 1)), params, [1 - 3 * 2.0 ** -24] * 2)


def test_sum_of_small_weights_of_the_bin_of_the_cut(vsl, H, dev):
    """20000 of 30000 tokens of 0.6 2^-42 of the largest, whose share is 2.7e-9 together."""
    V = 32768
    logits = row(V, (slice(0, 30000), np.log(0.6) - 42 * np.log(2)), (30000, 0))
    base.check(vsl, H, dev, logits[None], [(1.0, 20001, 1.0, 0.0)], [3.5e-9])


@pytest.mark.parametrize("V,spread", [(3000, 2.5), (50000, 2.5), (262147, 4.0)])
def test_broad_rows_too_large_for_bins(vsl, H, dev, V, spread):
    rng = np.random.default_rng(V)
    params = [(1.0, 0, 0.9, 0.0), (0.9, 5000 if V > 5000 else 700, 1.0, 0.0), (1.1, 1000, 0.95, 0.001), (1.0, 0, 0.999, 0.0),
              (0.7, 40, 0.9, 0.0), (1.0, 0, 1.0, 0.01)]
    logits = (20000 + rng.normal(0, spread, (len(params), V))).astype(np.float32)
    base.check(vsl, H, dev, logits, params, rng.random(len(params)))


def masked(logits, allowed, value):
    x = np.full_like(logits, value)
    x[allowed] = logits[allowed]
    return x


@pytest.mark.parametrize("V,dt", [(700, np.float32), (9001, np.float16), (32000, np.float32), (131072, np.float32)])
def test_finite_masks_are_masks(vsl, H, dev, V, dt):
    """Masks of finite values, among them the type's lowest, give what -infinity gives: with fewer tokens allowed than k, in some slices
    none; side by side and far apart; the last rows have all tokens masked."""
    rng = np.random.default_rng(V)
    params = [(1.0, 40, 0.9, 0.0), (0.7, 128, 1.0, 0.0), (1.5, 5, 1.0, 0.05), (1.0, 200, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.0)]
    logits = rng.normal(0, 3, V).astype(dt)
    for n in (1, 20, 60, 600):
        for allowed in (rng.permutation(V)[:n], np.arange(V // 3, V // 3 + n) % V):
            want, base_share = base.run(vsl, H, dev, np.tile(masked(logits, allowed, -np.inf), (len(params), 1)), params, [0.61] * len(params))
            for value in (-1e4, -65504.0, *([] if dt == np.float16 else [-1e9, np.finfo(np.float32).min])):
                x = np.tile(masked(logits, allowed, value), (len(params), 1))
                tok, share = base.run(vsl, H, dev, x, params, [0.61] * len(params))
                assert np.array_equal(tok, want) and np.all(np.abs(share - base_share) <= 2.0 ** -23 * base_share), (n, value)
                base.check(vsl, H, dev, x, params, rng.random(len(params)))
    x = np.full((len(params), V), np.finfo(dt).min, dt)
    tok, _ = base.run(vsl, H, dev, x, params, [0.0] * len(params))
    assert not tok.any()


def fastest(H, vsl, dev, logits, params):
    """The shortest of nine times of 20 calls, in ms."""
    torch, (rows, V) = dev.torch, logits.shape
    n = H.vsl_sample_rows_ws_bytes(rows, V)
    ws, par, u = dev.empty((n,), np.uint8), dev.put(base.structs(params)), dev.put(np.full(rows, 0.4, np.float32))
    tok, l, took = dev.empty((rows,), np.int32), dev.put(logits), []
    for _ in range(9):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(20):
            vsl.check(H.vsl_sample_rows(dev.p(l), 0, rows, V, V, dev.p(par), dev.p(u), dev.p(tok), None, dev.p(ws), n, None))
        b.record()
        dev.sync()
        took.append(a.elapsed_time(b))
    return min(took)


def test_cost_of_a_finite_mask(vsl, H, dev):
    """A step with 20 tokens allowed takes about as long with a finite mask as with -infinity: 2.6 times, where it took 48 times as
    long when the masked tokens counted among the k largest."""
    rng = np.random.default_rng(5)
    allowed, logits = rng.permutation(32000)[:20], rng.normal(0, 2.5, 32000).astype(np.float32)
    times = [fastest(H, vsl, dev, masked(logits, allowed, v)[None], [(0.7, 40, 0.9, 0.0)]) for v in (-np.inf, -1e9, np.finfo(np.float32).min)]
    assert max(times[1:]) < 8 * times[0], times


@pytest.mark.parametrize("rows,V", [(1, 32000), (1, 131072), (16, 131072), (64, 32000)])
def test_cost_of_a_larger_k(vsl, H, dev, rows, V):
    """A row with k up to 128, whose tokens come from the slices' lists, takes no longer than one with k = 200, which is cut by bins
    (7 to 35 times as long when the lists together held more than 1024 tokens)."""
    logits = np.random.default_rng(V).normal(0, 2.5, (rows, V)).astype(np.float32)
    times = [fastest(H, vsl, dev, logits, [(0.7, k, 0.9, 0.0)] * rows) for k in (200, 40, 64, 100, 128)]
    assert max(times[1:]) < 3 * times[0], times


@pytest.mark.parametrize("rows,V", [(1, 32000), (3, 50000), (1, 131072), (16, 131072), (2, 1 << 20)])
def test_long_lists(vsl, H, dev, rows, V):
    """k up to 128 from few and many slices, with ties where the lists end."""
    rng = np.random.default_rng(rows + V)
    for k in (40, 64, 100, 127, 128):
        for step in (0.0, 0.25):
            logits = rng.normal(0, 2.5, (rows, V)).astype(np.float32)
            if step:
                logits = (np.round(logits / step) * step).astype(np.float32)
            base.check(vsl, H, dev, logits, [(0.9, k, 0.95, 0.0)] * rows, rng.random(rows))
