"""Scaled rotary tables and the append with rotation of part of each head, against 64-bit definitions.

Tolerances (u = 2^-24, half a step of fp32; fp16 2^-11, subnormals 2^-25 absolute):
  tables    angles in 64 bits: frequencies within a few 2^-52 of theirs, positions below 2^20, so angles within 2^-29,
            15 rotations add 15 2^-51; each entry is rounded once: u |scale| + 2^-29 |scale|
  q, k      two products and a sum: 2 u (|a| + |b|) at most, taken as 3, then the output's rounding"""
import ctypes
import math

import numpy as np
import pytest

import token_step_ref as ref
import vsl_testlib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


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


SCALINGS = [dict(type=0), dict(type=1, factor=4.0), dict(type=2, factor=8.0, orig_ctx=8192.0, low=1.0, high=4.0),
            dict(type=3, factor=16.0, orig_ctx=4096.0, low=1.0, high=32.0),
            dict(type=3, factor=0.5, orig_ctx=100.0, low=0.5, high=300.0), dict(type=0, mscale=1.5)]


@pytest.mark.parametrize("scaling", range(len(SCALINGS)))
@pytest.mark.parametrize("rot,pos0,rows", [(128, 0, 700), (2, 0, 1), (10, 999983, 33), (20, 4097, 17), (130, 5, 15)])
def test_tables(vsl, H, dev, scaling, rot, pos0, rows):
    kw = SCALINGS[scaling]
    rng = np.random.default_rng(rot + rows + scaling)
    ff = (1 + rng.random(rot // 2) * 3).astype(np.float32) if scaling % 2 else None
    theta = 500000.0 if scaling == 2 else 10000.0
    s = vsl.RopeScaling(theta=theta, **kw)
    half = rot // 2
    cos, sin = (dev.put(np.full((rows + 1) * half, 7, np.float32)) for _ in range(2))
    fd = None if ff is None else dev.put(ff)
    vsl.check(H.vsl_rope_tables(rot, pos0, rows, ctypes.byref(s), dev.p(fd), dev.p(cos), dev.p(sin), None))
    f = ref.rope_freqs(rot, theta, kw["type"], kw.get("factor", 1.0), kw.get("orig_ctx", 0.0), kw.get("low", 0.0),
                       kw.get("high", 0.0), ff)
    m = kw.get("mscale") or (0.1 * math.log(kw["factor"]) + 1 if kw["type"] == 3 and kw["factor"] > 1 else 1.0)
    a = np.arange(pos0, pos0 + rows)[:, None] * f
    for got, want in ((dev.get(cos), np.cos(a) * m), (dev.get(sin), np.sin(a) * m)):
        assert np.all(np.abs(got[:rows * half].reshape(rows, half) - want) <= (U + 2.0 ** -29) * m * 1.01)
        assert np.all(got[rows * half:] == 7)  # nothing behind the last row


def _close(got, want, pair, dt):
    a = np.abs(want)
    last = 0.0 if dt == 0 else np.maximum(2.0 ** -11 * a, 2.0 ** -25) if dt == 1 else 2.0 ** -22 * a + 2.0 ** -25
    return np.all(np.abs(got - want) <= (3 * U * pair + last) * 1.001)


# n_q, n_kv, head_dim, rotated dims: whole heads, parts, odd halves, none; head dims other than attention's
SHAPES = [(4, 4, 64, 64), (6, 2, 128, 32), (8, 1, 80, 20), (3, 3, 8, 6), (32, 8, 128, 128), (5, 5, 96, 10), (2, 1, 512, 256),
          (4, 2, 64, 0)]


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("S,pos0,qdt,kvdt,given", [(1, 0, 0, 0, False), (37, 5, 2, 1, True), (130, 61, 1, 1, False)])
def test_append(vsl, H, dev, shape, halves, S, pos0, qdt, kvdt, given):
    nq, nkv, hd, rot = shape
    cap, table = pos0 + S + 3, 400
    rng = np.random.default_rng(S * 7 + hd + rot)
    qkv = rng.normal(0, 1.3, (S, nq + 2 * nkv, hd)).astype(np.float32)
    at = rng.integers(0, table, S).astype(np.uint32) if given else (pos0 + np.arange(S)).astype(np.uint32)
    ang = np.arange(table)[:, None] * ref.rope_freqs(max(rot, 2), 1e4)
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    kt = np.float16 if kvdt else np.float32
    kc, vc = (np.full((nkv, cap, hd), 3, kt) for _ in range(2))
    d = [dev.put(a) for a in (qkv, at, cos, sin, kc, vc)]
    q = dev.empty((2 if qdt == 2 else 1, S, nq, hd), np.float32 if qdt == 0 else np.float16)
    vsl.check(H.vsl_rope_part_append(dev.p(d[0]), S, nq, nkv, hd, rot, int(halves), pos0, dev.p(d[1]) if given else None,
                                     dev.p(d[2]), dev.p(d[3]), table, dev.p(q), qdt, dev.p(d[4]), dev.p(d[5]), kvdt, cap, None))
    want, pair = ref.rotate(qkv[:, :nq + nkv], cos[at][:, None, :rot // 2].astype(np.float64),
                            sin[at][:, None, :rot // 2].astype(np.float64), rot, halves)
    assert _close(dev.get(q).astype(np.float64).sum(0), want[:, :nq], pair[:, :nq], qdt)
    gk, gv = dev.get(d[4]).astype(np.float64), dev.get(d[5]).astype(np.float64)
    assert _close(gk[:, pos0:pos0 + S], want[:, nq:].transpose(1, 0, 2), pair[:, nq:].transpose(1, 0, 2), kvdt)
    v = qkv[:, nq + nkv:].transpose(1, 0, 2)
    assert np.array_equal(gv[:, pos0:pos0 + S], v.astype(kt).astype(np.float64))
    for c in (gk, gv):  # the other positions keep what they held
        assert np.all(c[:, :pos0] == 3) and np.all(c[:, pos0 + S:] == 3)


@pytest.mark.parametrize("shape", SHAPES[:6])
@pytest.mark.parametrize("kvdt", [0, 1])
def test_append_decode(vsl, H, dev, shape, kvdt):
    """One row at ctrl->pos: the bits of the row form; with a rotary position of its own; done and full caches."""
    nq, nkv, hd, rot = shape
    cap = table = 64
    rng = np.random.default_rng(hd)
    qkv = dev.put(rng.normal(0, 1, (nq + 2 * nkv) * hd).astype(np.float32))
    ang = np.arange(table)[:, None] * ref.rope_freqs(max(rot, 2), 1e4)
    cos, sin = dev.put(np.cos(ang).astype(np.float32)), dev.put(np.sin(ang).astype(np.float32))
    kt = np.float16 if kvdt else np.float32

    def caches():
        return [dev.put(np.full((nkv, cap, hd), 3, kt)) for _ in range(2)]

    for pos, own in ((0, None), (63, None), (17, 42)):
        where = None if own is None else dev.put(np.array([own], np.uint32))
        a, b = caches(), caches()
        q1, q2 = dev.empty((nq * hd,), np.float32), dev.empty((nq * hd,), np.float32)
        ctrl = dev.put(np.array([pos, 0, 0, 0, 9, 0, cap, 0], np.uint32))
        for halves in (0, 1):
            vsl.check(H.vsl_rope_part_append_decode(dev.p(qkv), nq, nkv, hd, rot, halves, dev.p(where), dev.p(cos), dev.p(sin),
                                                    table, dev.p(q1), dev.p(a[0]), dev.p(a[1]), kvdt, cap, dev.p(ctrl), None))
            vsl.check(H.vsl_rope_part_append(dev.p(qkv), 1, nq, nkv, hd, rot, halves, pos, dev.p(where), dev.p(cos), dev.p(sin),
                                             table, dev.p(q2), 0, dev.p(b[0]), dev.p(b[1]), kvdt, cap, None))
            assert np.array_equal(dev.get(q1), dev.get(q2))
            assert all(np.array_equal(dev.get(x), dev.get(y)) for x, y in zip(a, b))
    for pos, done in ((5, 1), (64, 0), (0xFFFFFFFF, 0)):
        c = caches()
        q = dev.put(np.full(nq * hd, 9, np.float32))
        ctrl = dev.put(np.array([pos, 0, done, 0, 9, 0, cap, 0], np.uint32))
        vsl.check(H.vsl_rope_part_append_decode(dev.p(qkv), nq, nkv, hd, rot, 0, None, dev.p(cos), dev.p(sin), table, dev.p(q),
                                                dev.p(c[0]), dev.p(c[1]), kvdt, cap, dev.p(ctrl), None))
        assert np.all(dev.get(q) == 9) and all(np.all(dev.get(x) == 3) for x in c)
        after = dev.get(ctrl, np.uint32)
        assert after[2] == 1 and after[7] == (0 if done else 1)


@pytest.mark.parametrize("rot", [64, 20])
@pytest.mark.parametrize("halves", [0, 1])
def test_positions_past_the_tables(vsl, H, dev, rot, halves):
    """Rotated dims of such a row are NaN, its other dims and the other rows are not."""
    nq, nkv, hd, S, table = 2, 1, 64, 3, 16
    x = np.ones((S, nq + 2 * nkv, hd), np.float32)
    at = dev.put(np.array([15, 16, 0xFFFFFFFF], np.uint32))
    ang = np.arange(table)[:, None] * ref.rope_freqs(rot, 1e4)
    cos, sin = dev.put(np.cos(ang).astype(np.float32)), dev.put(np.sin(ang).astype(np.float32))
    kc, vc, q = (dev.empty(s, np.float32) for s in ((nkv, S, hd), (nkv, S, hd), (S, nq, hd)))
    xd = dev.put(x)
    vsl.check(H.vsl_rope_part_append(dev.p(xd), S, nq, nkv, hd, rot, halves, 0, dev.p(at), dev.p(cos), dev.p(sin), table,
                                     dev.p(q), 0, dev.p(kc), dev.p(vc), 0, S, None))
    for got in (dev.get(q), dev.get(kc).transpose(1, 0, 2)):
        assert np.all(np.isfinite(got[0])) and np.all(np.isnan(got[1:, :, :rot])) and np.all(got[1:, :, rot:] == 1)
    assert np.all(dev.get(vc) == 1)
