"""Attention over the 4-bit KV cache where its kernels hand data from wave to wave, read what no append wrote, or add a
long tail of small probabilities. Definitions: kv4_ref; tolerances: those of test_kv4_gpu, unless a test states its own."""
import math

import numpy as np
import pytest

import kv4_ref
from test_kv4_gpu import H, _dev, attn_tol, dev, filled, out_tol, prefill  # noqa: F401 (fixtures)

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
