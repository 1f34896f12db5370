"""Limits of attention with modified scores that the host checks: workspace sizes, which never divide by zero and never exceed
what serves every call, and caps."""
import ctypes
import random

import pytest


@pytest.fixture(scope="module")
def ws(vsl):
    return vsl.hip().vsl_attn_prefill_mods_ws_bytes


@pytest.mark.parametrize("S,pos0,n_q,n_kv", [(0xFFFFFFFF, 0, 8, 2), (0xFFFFFFE1, 7, 1, 1), (0x80000000, 0, 256, 256),
                                             (0x80000000, 0xFFFFFFFF, 1 << 31, 1 << 31), (0xFFFFFFFF, 0xFFFFFFFF, 0xFFFFFFFF, 1),
                                             (0xFFFFFFE0, 0, 0xFFFFFFFF, 0xFFFFFFFF)])
def test_sizes_that_no_call_takes(ws, S, pos0, n_q, n_kv):
    """A number of blocks that does not fit 32 bits is many blocks, not none."""
    assert ws(S, pos0, n_q, n_kv, 128) == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_one_size_serves_every_call(vsl, ws, hd):
    rng = random.Random(hd)
    most, some = vsl.ATTN_MODS_WS_MAX(hd), 0
    for n_kv in (1, 2, 3, 8, 40, 256, 1000):
        for g in range(1, 9):
            for _ in range(200):
                S, pos0 = int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 24))
                n = ws(S, pos0, n_kv * g, n_kv, hd)
                assert n <= most, (S, pos0, n_kv * g, n_kv)
                some = max(some, n)
    assert some > most // 2


def test_factors_below_the_normal_numbers_are_refused(vsl):
    """scale / softcap and softcap * log2(e) would lose digits."""
    H = vsl.hip()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) & ~255
    for scale, cap in ((0.09, 2e38), (-0.09, 2e38), (1e-20, 1e19), (1e-38, 2e38), (1e-45, 1.0), (1e-40, 1e-40), (1e-39, 7e-39)):
        m = ctypes.byref(vsl.AttnMods(softcap=cap))
        assert H.vsl_attn_prefill_mods(p, 1, p, p, 4, 0, 8, 2, 128, 64, scale, p, 1, m, None, 0, None) == -100, (scale, cap)
        assert H.vsl_attn_decode_mods(p, p, p, 1, 8, 2, 128, 64, scale, 4, p, p, p, p, m, None) == -100, (scale, cap)
