"""Sampling of rows where weights are far apart: rows whose small weights add up.

Tolerances: tokens are equal, u lying further than 1e-10 from every border; a share is one fp32 rounding (2^-24) off, and 1e-10."""
import numpy as np
import pytest

import test_sample_rows_gpu as base
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
