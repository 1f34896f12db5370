"""The 4-bit KV cache without a GPU: its sizes, and the calls that are refused before anything is launched."""
import ctypes

import numpy as np
import pytest

import kv4_ref


@pytest.fixture(scope="module")
def H(vsl):
    return vsl.hip()


def ptr(n=4096, off=0):
    """An address that no refused call reads."""
    return 1 << 20 | off


def test_cache_bytes(vsl, H):
    for n_kv, cap, hd in [(1, 1, 64), (8, 4096, 128), (3, 1000, 64), (8, 128, 128), (8, 129, 128), (2, 40000000, 128)]:
        assert H.vsl_kv_cache_bytes(vsl.VSL_DT_KV4, n_kv, cap, hd) == kv4_ref.cache_bytes(n_kv, cap, hd)
        assert H.vsl_kv_cache_bytes(vsl.VSL_DT_F16, n_kv, cap, hd) == 2 * n_kv * cap * hd
        assert H.vsl_kv_cache_bytes(vsl.VSL_DT_F32, n_kv, cap, hd) == 4 * n_kv * cap * hd
    # 4.5 bits a value
    assert H.vsl_kv_cache_bytes(vsl.VSL_DT_KV4, 8, 32768, 128) == 8 * 32768 * 128 * 9 // 16
    for dt, hd in [(vsl.VSL_DT_KV4, 96), (vsl.VSL_DT_KV4, 256), (vsl.VSL_DT_F16X2, 128), (99, 128)]:
        assert H.vsl_kv_cache_bytes(dt, 8, 128, hd) == 0


def _append(vsl, H, **kw):
    a = dict(qkv=ptr(), S=3, nq=4, nkv=2, hd=64, pos0=0, gq=ptr(), gk=ptr(), eps=1e-5, rope=0, cos=ptr(), sin=ptr(), q=ptr(),
             qdt=vsl.VSL_DT_F32, kc=ptr(), vc=ptr(), kvdt=vsl.VSL_DT_KV4, cap=64)
    a.update(kw)
    return H.vsl_qk_norm_rope_append(*a.values(), None)


def _append_decode(vsl, H, **kw):
    a = dict(qkv=ptr(), nq=4, nkv=2, hd=64, gq=ptr(), gk=ptr(), eps=1e-5, rope=0, cos=ptr(), sin=ptr(), q=ptr(), kc=ptr(),
             vc=ptr(), kvdt=vsl.VSL_DT_KV4, cap=64, ctrl=ptr())
    a.update(kw)
    return H.vsl_qk_norm_rope_append_decode(*a.values(), None)


REFUSED = [(dict(qkv=None), -100), (dict(cos=None), -100), (dict(sin=None), -100), (dict(q=None), -100), (dict(kc=None), -100),
           (dict(vc=None), -100), (dict(hd=96), -103), (dict(hd=256), -103), (dict(nq=0), -100), (dict(nkv=0), -100),
           (dict(rope=2), -100), (dict(rope=-1), -100), (dict(kvdt=2), -103), (dict(kvdt=5), -103), (dict(cap=0), -100),
           (dict(qkv=ptr(off=4)), -100), (dict(gq=ptr(off=8)), -100), (dict(gk=ptr(off=4)), -100), (dict(cos=ptr(off=4)), -100),
           (dict(sin=ptr(off=8)), -100), (dict(q=ptr(off=8)), -100), (dict(kc=ptr(off=16)), -100), (dict(vc=ptr(off=128)), -100),
           (dict(kc=ptr(off=8), kvdt=1), -100), (dict(nq=0x7FFFFFFF), -100)]


@pytest.mark.parametrize("kw,code", REFUSED, ids=[str(k) for k, _ in REFUSED])
def test_append_refusals(vsl, H, kw, code):
    assert _append(vsl, H, **kw) == code
    assert H.vsl_last_error().decode().startswith("vsl_qk_norm_rope_append")
    assert _append_decode(vsl, H, **kw) == code


def test_append_refusals_of_one_entry(vsl, H):
    assert _append(vsl, H, qdt=vsl.VSL_DT_F16F8) == -103
    assert _append(vsl, H, pos0=62) == -104
    assert _append(vsl, H, pos0=0xFFFFFFFF) == -104
    assert _append(vsl, H, S=65) == -104
    assert _append(vsl, H, S=0) == 0
    assert _append_decode(vsl, H, ctrl=None) == -100
    # more values than a launch has lanes for
    assert _append(vsl, H, S=1 << 26, nq=32, nkv=8, hd=128, cap=1 << 27) == -103
    assert _append(vsl, H, S=0xFFFFFFFF, nq=1, nkv=1, hd=128, cap=0xFFFFFFFF) == -103


def test_read_refusals(vsl, H):
    def read(kc=ptr(), vc=ptr(), nkv=2, cap=64, hd=64, pos0=0, n=3, ko=ptr(), vo=ptr(), dt=1):
        return H.vsl_kv4_read(kc, vc, nkv, cap, hd, pos0, n, ko, vo, dt, None)

    assert read(n=0) == 0
    for kw in (dict(kc=None), dict(vo=None), dict(kc=None, ko=None, vc=None, vo=None), dict(nkv=0), dict(kc=ptr(off=64)),
               dict(ko=ptr(off=8))):
        assert read(**kw) == -100, kw
    assert read(hd=32) == -103
    assert read(dt=2) == -103
    assert read(nkv=8, hd=128, n=1 << 27, cap=1 << 28) == -103
    assert read(pos0=62) == -104
    assert read(pos0=0xFFFFFFFF, n=2) == -104


def test_attention_refusals(vsl, H):
    def prefill(q=ptr(), qdt=1, kc=ptr(), vc=ptr(), S=4, pos0=0, nq=8, nkv=2, hd=128, cap=64, out=ptr(), odt=1, win=None):
        a = (q, qdt, kc, vc, S, pos0, nq, nkv, hd, cap, 0.1, out, odt)
        if win:
            return H.vsl_attn_prefill_kv4_window(*a, *win, None)
        return H.vsl_attn_prefill_kv4(*a, None)

    assert prefill(S=0) == 0
    for kw in (dict(q=None), dict(kc=None), dict(out=None), dict(nkv=0), dict(nq=0), dict(nq=7), dict(kc=ptr(off=16)),
               dict(q=ptr(off=8)), dict(out=ptr(off=2)), dict(win=(0x7FFFFFFF, 1, 8))):
        assert prefill(**kw) == -100, kw
    for kw in (dict(hd=96), dict(nq=18), dict(qdt=0), dict(odt=0), dict(qdt=3)):
        assert prefill(**kw) == -103, kw
    assert prefill(pos0=61) == -104
    assert prefill(S=1 << 24, cap=1 << 25) == -103

    def decode(kc=ptr(), vc=ptr(), nq=8, nkv=2, hd=128, cap=64, nsplit=4, dt=vsl.VSL_DT_KV4):
        return H.vsl_attn_decode(ptr(), kc, vc, dt, nq, nkv, hd, cap, 0.1, nsplit, ptr(), ptr(), ptr(), ptr(), None)

    assert decode(kc=ptr(off=32)) == -100
    assert decode(cap=0) == -100
    assert decode(nq=7) == -100
    assert decode(nsplit=0) == -100
    assert decode(nq=18) == -103
    assert decode(hd=32) == -103
    for q, po, ml in [(ptr(off=8), ptr(), ptr()), (ptr(), ptr(off=8), ptr()), (ptr(), ptr(), ptr(off=4))]:
        assert H.vsl_attn_decode(q, ptr(), ptr(), vsl.VSL_DT_KV4, 8, 2, 128, 64, 0.1, 4, po, ml, ptr(), ptr(), None) == -100
    # the fused projection writes fp16 and fp32 caches only
    assert H.vsl_qkv_rope_append(ptr(), ptr(), 1e-5, ptr(), 1, 256, 4, 4, 64, ptr(), ptr(), ptr(), ptr(), vsl.VSL_DT_KV4, 64,
                                 ptr(), ptr(), None) == -103


def test_norm_gemv_refusals(vsl, H):
    assert H.vsl_norm_gemv(None, ptr(), 1e-5, ptr(), 1, 64, 64, ptr(), None, None) == -100
    assert H.vsl_norm_gemv(ptr(), ptr(), 1e-5, ptr(), 1, 0, 64, ptr(), None, None) == -100
    assert H.vsl_norm_gemv(ptr(), ptr(), 1e-5, ptr(), 1, 64, 63, ptr(), None, None) == -100
    assert H.vsl_norm_gemv(ptr(), ptr(), 1e-5, ptr(), 99, 64, 64, ptr(), None, None) == -103


def test_reference_form():
    """The reference itself: every value within half a step, exact in binary16; a pack reads back."""
    rng = np.random.default_rng(0)
    for std in (1e-6, 1e-3, 1.0, 50.0, 8000.0):
        x = rng.normal(0, std, (2, 40, 64))
        codes, steps = kv4_ref.quantize(x)
        v = kv4_ref.values(codes, steps)
        d = (steps & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64)
        assert np.all(np.abs(v - x).reshape(2, 40, 2, 32) <= d[..., None] / 2 * (1 + 1e-12))
        assert np.array_equal(v.astype(np.float16).astype(np.float64), v)
        for is_v in (False, True):
            buf = rng.integers(0, 256, kv4_ref.cache_bytes(2, 50, 64), dtype=np.uint8)
            kv4_ref.pack(buf, x, 5, 2, 50, 64, is_v)
            assert np.array_equal(kv4_ref.unpack(buf, 5, 40, 2, 50, 64, is_v), v)
