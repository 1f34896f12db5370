"""Refusals of scaled rotation, partial rotation, attention with modified scores and sampling of rows: everything that the
host can see is refused before a launch, so this runs without a GPU."""
import ctypes

import numpy as np
import pytest

import token_step_ref as ref

BUF = (ctypes.c_char * 8192)()
BASE = (ctypes.addressof(BUF) + 255) & ~255


def ptr(off=0):
    return BASE + off


@pytest.fixture(scope="module")
def H(vsl):
    return vsl.hip()


def test_rope_tables(vsl, H):
    def call(rot=64, pos0=0, rows=4, ff=None, cos=ptr(), sin=ptr(), null=False, **kw):
        s = dict(type=0, theta=1e4, factor=4.0, orig_ctx=4096.0, low=1.0, high=4.0, mscale=0.0)
        s.update(kw)
        return H.vsl_rope_tables(rot, pos0, rows, None if null else ctypes.byref(vsl.RopeScaling(**s)), ff, cos, sin, None)

    inf, nan = float("inf"), float("nan")
    assert call(rows=0) == 0
    for kw in (dict(null=True), dict(cos=None), dict(sin=None), dict(theta=0.0), dict(theta=-1.0), dict(theta=inf),
               dict(theta=nan), dict(mscale=-1.0), dict(mscale=nan), dict(type=1, factor=0.0), dict(type=1, factor=nan),
               dict(type=2, low=4.0, high=4.0), dict(type=2, low=0.0), dict(type=2, orig_ctx=0.0), dict(type=3, high=nan),
               dict(type=3, theta=1.0), dict(cos=ptr(2)), dict(ff=ptr(1))):
        assert call(**kw) == -100, kw
    for kw in (dict(rot=0), dict(rot=63), dict(rot=514), dict(type=4), dict(type=-1), dict(pos0=0xFFFFFFFF),
               dict(pos0=1 << 31, rows=1)):
        assert call(**kw) == -103, kw


def test_append(vsl, H):
    def call(qkv=ptr(), S=2, nq=8, nkv=2, hd=128, rot=64, rope=0, pos0=0, positions=None, cos=ptr(), sin=ptr(), rows=64,
             q=ptr(), qdt=0, kc=ptr(), vc=ptr(), kvdt=1, cap=64):
        return H.vsl_rope_part_append(qkv, S, nq, nkv, hd, rot, rope, pos0, positions, cos, sin, rows, q, qdt, kc, vc, kvdt,
                                      cap, None)

    def step(ctrl=ptr(), rot=64, q=ptr(), nq=8, cos=ptr(), kvdt=1):
        return H.vsl_rope_part_append_decode(ptr(), nq, 2, 128, rot, 0, None, cos, ptr(), 64, q, ptr(), ptr(), kvdt, 64, ctrl,
                                             None)

    assert call(S=0) == 0
    assert call(S=0, rot=0, cos=None, sin=None, rows=0) == 0
    for kw in (dict(qkv=None), dict(cos=None), dict(sin=None), dict(q=None), dict(kc=None), dict(vc=None), dict(rot=63),
               dict(rot=130), dict(nq=0), dict(nkv=0), dict(rope=2), dict(cap=0), dict(rows=0), dict(qkv=ptr(8)), dict(q=ptr(8)),
               dict(cos=ptr(4)), dict(kc=ptr(2)), dict(positions=ptr(2)), dict(nq=0xFFFFFFFF)):
        assert call(**kw) == -100, kw
    for kw in (dict(hd=0, rot=0), dict(hd=100, rot=0), dict(hd=520), dict(qdt=3), dict(kvdt=2), dict(kvdt=7),
               dict(S=1 << 24, cap=1 << 25)):
        assert call(**kw) == -103, kw
    assert call(pos0=63) == -104
    assert call(pos0=0xFFFFFFFF) == -104
    for kw in (dict(ctrl=None), dict(rot=63), dict(q=None), dict(q=ptr(4)), dict(nq=0), dict(cos=None)):
        assert step(**kw) == -100, kw
    assert step(kvdt=7) == -103


def _mods(vsl, **kw):
    return ctypes.byref(vsl.AttnMods(**{**dict(softcap=0.0, slopes=None, ranges=None), **kw}))


def test_decode_attention(vsl, H):
    def call(q=ptr(), kc=ptr(), vc=ptr(), kvdt=1, nq=8, nkv=2, hd=128, cap=64, nsplit=4, po=ptr(), pml=ptr(), out=ptr(),
             ctrl=ptr(), **mods):
        return H.vsl_attn_decode_mods(q, kc, vc, kvdt, nq, nkv, hd, cap, 0.1, nsplit, po, pml, out, ctrl, _mods(vsl, **mods),
                                      None)

    for kw in (dict(q=None), dict(kc=None), dict(vc=None), dict(po=None), dict(pml=None), dict(out=None), dict(ctrl=None),
               dict(nkv=0), dict(nq=0), dict(nq=7), dict(cap=0), dict(cap=0x80000000), dict(nsplit=0), dict(nsplit=1025),
               dict(q=ptr(4)), dict(kc=ptr(8)), dict(po=ptr(4)), dict(pml=ptr(4)), dict(out=ptr(8)), dict(softcap=-1.0),
               dict(softcap=float("nan")), dict(softcap=float("inf")), dict(softcap=3e38), dict(softcap=1e-40), dict(slopes=ptr(2)),
               dict(ranges=ptr(4))):
        assert call(**kw) == -100, kw
    for kw in (dict(nq=18), dict(hd=96), dict(kvdt=7), dict(kvdt=2)):
        assert call(**kw) == -103, kw


def test_prompt_attention(vsl, H):
    def call(q=ptr(), qdt=1, kc=ptr(), vc=ptr(), S=4, pos0=0, nq=8, nkv=2, hd=128, cap=64, out=ptr(), odt=1, ws=None, n=0,
             **mods):
        return H.vsl_attn_prefill_mods(q, qdt, kc, vc, S, pos0, nq, nkv, hd, cap, 0.1, out, odt, _mods(vsl, **mods), ws, n, None)

    assert call(S=0) == 0
    for kw in (dict(q=None), dict(kc=None), dict(vc=None), dict(out=None), dict(nkv=0), dict(nq=0), dict(nq=7), dict(q=ptr(8)),
               dict(out=ptr(8)), dict(kc=ptr(8)), dict(ws=ptr(8)), dict(cap=0x80000000), dict(softcap=-1.0), dict(slopes=ptr(1)),
               dict(ranges=ptr(4)), dict(softcap=3e38), dict(softcap=1e-40), dict(softcap=float("inf"))):
        assert call(**kw) == -100, kw
    for kw in (dict(nq=65536, nkv=8192), dict(nq=18), dict(hd=96), dict(qdt=0), dict(odt=0), dict(qdt=3), dict(S=1 << 24, cap=1 << 25)):
        assert call(**kw) == -103, kw
    assert call(pos0=61) == -104
    assert call(pos0=0xFFFFFFFF) == -104
    ws = H.vsl_attn_prefill_mods_ws_bytes
    assert ws(0, 0, 8, 2, 128) == ws(4, 0, 8, 0, 128) == ws(4, 0, 7, 2, 128) == ws(4, 0, 8, 2, 96) == 0
    assert ws(4096, 0, 32, 8, 128) == 0  # enough blocks of rows
    assert ws(1, 30000, 8, 2, 128) >= 2 * 8 * 130 * 4


def test_sample_rows(vsl, H):
    need = H.vsl_sample_rows_ws_bytes(3, 500)
    assert need > 0

    def call(logits=ptr(), dt=0, rows=3, V=500, stride=500, params=ptr(), u=ptr(), tokens=ptr(), probs=ptr(), ws=ptr(), n=need):
        return H.vsl_sample_rows(logits, dt, rows, V, stride, params, u, tokens, probs, ws, n, None)

    assert call(rows=0) == 0
    for kw in (dict(logits=None), dict(params=None), dict(u=None), dict(tokens=None), dict(ws=None), dict(stride=499),
               dict(ws=ptr(8)), dict(logits=ptr(2)), dict(dt=1, logits=ptr(1)), dict(params=ptr(2)), dict(u=ptr(1)),
               dict(tokens=ptr(2)), dict(probs=ptr(2))):
        assert call(**kw) == -100, kw
    for kw in (dict(dt=2), dict(V=0, stride=0), dict(V=(1 << 20) + 1, stride=1 << 21), dict(rows=65536)):
        assert call(**kw) == -103, kw
    assert call(n=need - 1) == -104
    assert H.vsl_sample_rows_ws_bytes(0, 5) == H.vsl_sample_rows_ws_bytes(5, 0) == H.vsl_sample_rows_ws_bytes(1, (1 << 20) + 1) == 0


def test_definitions():
    """The reference itself: scalings by hand at their ends, and the cuts of a row small enough to count."""
    f = ref.rope_freqs(64, 1e4)
    assert np.allclose(ref.rope_freqs(64, 1e4, 1, 4.0), f / 4)
    turns = ref.rope_freqs(64, 1e4, 2, 8.0, 8192.0, 1.0, 4.0)
    n = 8192.0 * f / (2 * np.pi)
    assert np.array_equal(turns[n > 4], f[n > 4]) and np.allclose(turns[n < 1], f[n < 1] / 8)
    yarn = ref.rope_freqs(64, 1e4, 3, 16.0, 4096.0, 1.0, 32.0)
    assert yarn[0] == f[0] and np.isclose(yarn[-1], f[-1] / 16) and np.all(np.diff(yarn) < 0)
    l = np.log(np.array([1.0, 4.0, 2.0, 2.0, 1.0]))  # weights 1/4, 1, 1/2, 1/2, 1/4
    assert ref.sample(l, 1.0, 0, 1.0, 0.0, 0.05)[0] == 0
    assert ref.sample(l, 1.0, 3, 1.0, 0.0, 0.99)[:2] == (3, pytest.approx(0.25))
    assert ref.sample(l, 1.0, 2, 1.0, 0.0, 0.99)[:2] == (2, pytest.approx(1 / 3))
    assert ref.sample(l, 1.0, 0, 0.7, 0.0, 0.99)[0] == 3     # 1 + 1/2 + 1/2 of 2.5 reach 0.7
    assert ref.sample(l, 1.0, 0, 0.6, 0.0, 0.99)[0] == 2     # 1 + 1/2 do
    assert ref.sample(l, 1.0, 0, 1.0, 0.3, 0.999)[0] == 3
    assert ref.sample(l, 0.0, 0, 1.0, 0.0, 0.5)[0] == 1
