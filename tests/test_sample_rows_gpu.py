"""Sampling of rows by temperature, top-k, top-p and min-p, against the definition in 64 bits: tokens are equal but where u
or the top-p cut lies within 1e-10 of a border (no seed here does); shares are one fp32 rounding (2^-24) off, plus 1e-10."""
import ctypes

import numpy as np
import pytest

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


def structs(params):
    """(temperature, top_k, top_p, min_p) rows as the device's structs."""
    a = np.zeros((len(params), 4), np.float32)
    for i, (t, k, p, m) in enumerate(params):
        a[i] = (t, 0, p, m)
        a[i, 1:2].view(np.uint32)[0] = k
    return a


def run(vsl, H, dev, logits, params, u, stride=None, want_probs=True, stream=None):
    rows, V = logits.shape
    stride = stride or V
    buf = np.full((rows, stride), np.inf, logits.dtype)  # what lies between the rows is not read
    buf[:, :V] = logits
    n = H.vsl_sample_rows_ws_bytes(rows, V)
    ws = dev.put(np.full(n, 0xA5, np.uint8))
    l, p, ud = dev.put(buf), dev.put(structs(params)), dev.put(np.asarray(u, np.float32))
    tok, pr = dev.put(np.full(rows + 1, 77, np.int32)), dev.put(np.full(rows + 1, 77, np.float32))
    dt = vsl.VSL_DT_F16 if logits.dtype == np.float16 else vsl.VSL_DT_F32
    vsl.check(H.vsl_sample_rows(dev.p(l), dt, rows, V, stride, dev.p(p), dev.p(ud), dev.p(tok), dev.p(pr) if want_probs else None,
                                dev.p(ws), n, stream))
    t, q = dev.get(tok), dev.get(pr)
    assert t[rows] == 77 and q[rows] == 77
    return t[:rows], q[:rows]


def check(vsl, H, dev, logits, params, u, **kw):
    tok, share = run(vsl, H, dev, logits, params, u, **kw)
    for r in range(len(params)):
        t, k, p, m = (float(np.float32(x)) for x in params[r])
        want, ws, near = ref.sample(logits[r].astype(np.float64), t, int(k), p, m, float(np.float32(u[r])))
        assert near > 1e-10
        assert tok[r] == want, (r, params[r], u[r])
        assert abs(float(share[r]) - ws) <= 2.0 ** -24 * ws * 1.001 + 1e-10, (r, params[r])


PARAMS = [(0.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (1.2, 0, 1.0, 0.05), (0.8, 200, 0.95, 0.02),
          (1.0, 0, 1.0, 0.0), (1.5, 1000, 0.8, 0.0), (0.3, 257, 1.0, 0.0), (2.0, 256, 0.5, 0.0), (1.0, 1, 0.5, 0.0),
          (1.0, 0, 0.999, 0.001), (5.0, 3000, 0.99, 0.3), (1.0, 2, 1.0, 0.0), (1.0, 0, 0.01, 0.0), (0.05, 500, 0.9, 0.0),
          (100.0, 0, 0.6, 0.0)]


@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("V,spread", [(1, 1.0), (2, 1.0), (63, 2.0), (1000, 1.0), (1025, 3.0), (4096, 2.5), (32000, 2.5),
                                      (40961, 0.5), (131072, 2.5), (262147, 4.0)])
def test_rows(vsl, H, dev, V, spread, dt):
    rng = np.random.default_rng(V)
    rows = len(PARAMS)
    logits = rng.normal(0, spread, (rows, V)).astype(dt)
    check(vsl, H, dev, logits, PARAMS, rng.random(rows), stride=V + 3)


@pytest.mark.parametrize("rows", [1, 2, 70])
def test_row_counts(vsl, H, dev, rows):
    """Slices of 2048, 4096 and 8192 tokens."""
    rng = np.random.default_rng(rows)
    V = 50000
    params = [PARAMS[(3 * i + 1) % len(PARAMS)] for i in range(rows)]
    check(vsl, H, dev, rng.normal(0, 2, (rows, V)).astype(np.float32), params, rng.random(rows), want_probs=True)


def test_most_slices(vsl, H, dev):
    rng = np.random.default_rng(9)
    V = 1 << 20
    params = [PARAMS[i] for i in (1, 2, 5, 6)]
    check(vsl, H, dev, rng.normal(0, 2, (4, V)).astype(np.float32), params, rng.random(4))


def test_ends_of_u(vsl, H, dev):
    """u of 0 takes the first kept token, the largest float below 1 (and 1, and above) the last whose share is not lost in
    u's own steps; NaN and negative ones count as 0."""
    V = 5000
    logits = np.zeros((6, V), np.float32)
    logits[:, 17] = 0.5
    u = [0.0, np.nan, -3.0, 1.0 - 2.0 ** -24, 1.0, np.inf]
    for p in ((1.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.9), (1.0, 300, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 20, 1.0, 0.0)):
        check(vsl, H, dev, logits, [p] * 6, u)


def test_ties(vsl, H, dev):
    """Constant rows and rows of few values: the order goes by index, lists overflow, cuts fall among equal logits."""
    rng = np.random.default_rng(3)
    V = 30011
    kinds = [np.zeros(V), np.full(V, -7.25), rng.integers(0, 2, V) * 1.0, rng.integers(0, 7, V) * 0.25 - 100,
             np.where(np.arange(V) % 3 == 0, 1e30, -1e30)]
    params = [(1.0, 40, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.2), (1.0, 5000, 0.7, 0.0), (1.0, 5000, 1.0, 0.0),
              (1.0, 7, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0)]
    for l in kinds:
        check(vsl, H, dev, np.tile(l.astype(np.float32), (len(params), 1)), params, rng.random(len(params)))


@pytest.mark.parametrize("V", [64, 4000, 8192, 30000])
def test_exact_borders(vsl, H, dev, V):
    """Equal logits: weights are whole numbers, so shares and draws that end on a border are exact."""
    params = [(1.0, 0, 0.5, 0.0), (1.0, 0, 0.25, 0.0), (0.7, V - 1, 0.5, 0.0), (1.0, 300, 0.75, 0.0), (1.0, 40, 0.5, 0.0),
              (1.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 1.0)]
    for value in (0.0, 3.3, -20.1):
        logits = np.full((len(params), V), value, np.float32)
        for u in (0.0, 0.5, 0.75):
            tok, _ = run(vsl, H, dev, logits, params, [u] * len(params))
            for r, (t, k, p, m) in enumerate(params):
                assert tok[r] == ref.sample(logits[r].astype(np.float64), t, k, p, m, u)[0], (value, u, params[r])


def test_masked_and_infinite(vsl, H, dev):
    """-infinity and NaN are never drawn, +infinity counts as the largest float, rows without a token give 0 with share 0."""
    rng = np.random.default_rng(4)
    V = 9001
    base = rng.normal(0, 2, V).astype(np.float32)
    few, low, nan, inf, none, nans, one = (base.copy() for _ in range(7))
    few[rng.permutation(V)[60:]] = -np.inf          # 60 tokens left
    low[rng.permutation(V)[500:]] = -3.4028235e38   # masked by the type's lowest value
    nan[::2] = np.nan
    inf[[77, 4000, 8999]] = np.inf
    none[:] = -np.inf
    nans[:] = np.nan
    one[:] = -np.inf
    one[5555] = -1e4
    params = [(1.0, 40, 0.9, 0.0), (1.0, 200, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.2), (1.0, 5000, 0.7, 0.0),
              (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0)]
    for l in (few, low, nan, inf, none, nans, one):
        check(vsl, H, dev, np.tile(l, (len(params), 1)), params, rng.random(len(params)))


def test_odd_parameters(vsl, H, dev):
    """NaN, negative, infinite and tiny parameters."""
    rng = np.random.default_rng(5)
    V, inf, nan = 6000, float("inf"), float("nan")
    l = rng.normal(0, 2, V).astype(np.float32)
    params = [(nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0), (1.0, 0, nan, nan), (1.0, 0, 0.0, 0.0), (1.0, 0, -2.0, 0.0),
              (1.0, 0, 1.0, 1.5), (1.0, 0, 1.0, 1.0), (1.0, 0, 2.0, -1.0), (1.0, 0xFFFFFFFF, 0.9, 0.0), (inf, 0, 1.0, 0.0),
              (inf, 0, 0.5, 0.0), (inf, 100, 1.0, 0.0), (1e-30, 0, 0.9, 0.0), (1e-3, 0, 0.9, 0.0), (1e-4, 0, 0.9, 0.0),
              (1e-30, 5, 1.0, 0.0), (1e-30, 0, 1.0, 0.0)]
    u = rng.random(len(params))
    tok, share = run(vsl, H, dev, np.tile(l, (len(params), 1)), params, u)
    for r, (t, k, p, m) in enumerate(params):
        t = 0.0 if np.isnan(t) else float(np.float32(t))
        p = 1.0 if np.isnan(p) else p
        m = 0.0 if np.isnan(m) else m
        if m > 1:
            t = 0.0
        want, ws, near = ref.sample(l.astype(np.float64), t, int(k), p, m, float(np.float32(u[r])))
        # (an infinite temperature makes whole numbers of the weights: borders that are met exactly are decided, too)
        assert (near > 1e-10 or t == inf) and tok[r] == want, (r, params[r])
        assert abs(float(share[r]) - ws) <= 2.0 ** -24 * ws * 1.001 + 1e-10, (r, params[r])


def test_graph_with_changing_parameters(vsl, H, dev):
    """A captured call serves the logits, parameters and numbers that its memory holds at each replay; two graphs that
    share a workspace, one after the other."""
    rng = np.random.default_rng(6)
    rows, V = 5, 20000
    n = H.vsl_sample_rows_ws_bytes(rows, V)
    ws = dev.empty((n,), np.uint8)
    torch = dev.torch
    sets = []
    for i in range(2):
        sets.append([dev.empty((rows, V), np.float32), dev.empty((rows, 4), np.float32), dev.empty((rows,), np.float32),
                     dev.empty((rows,), np.int32), dev.empty((rows,), np.float32)])
    s = ctypes.c_void_p()
    vsl.check(H.vsl_stream_create(ctypes.byref(s)))
    graphs = []
    dev.sync()
    for l, p, u, tok, pr in sets:
        g = ctypes.c_void_p()
        vsl.check(H.vsl_graph_begin(s))
        vsl.check(H.vsl_sample_rows(dev.p(l), 0, rows, V, V, dev.p(p), dev.p(u), dev.p(tok), dev.p(pr), dev.p(ws), n, s))
        vsl.check(H.vsl_graph_end(s, ctypes.byref(g)))
        graphs.append(g)
    for turn in range(4):
        held = []
        for i, (l, p, u, tok, pr) in enumerate(sets):
            lh = rng.normal(0, 2, (rows, V)).astype(np.float32)
            ph = [PARAMS[(turn * 5 + i * 3 + r) % len(PARAMS)] for r in range(rows)]
            uh = rng.random(rows).astype(np.float32)
            l.copy_(torch.from_numpy(lh))
            p.copy_(torch.from_numpy(structs(ph)))
            u.copy_(torch.from_numpy(uh))
            held.append((lh, ph, uh))
        dev.sync()
        for g in graphs:
            vsl.check(H.vsl_graph_launch(g, s))
        vsl.check(H.vsl_stream_sync(s))
        for (lh, ph, uh), (_, _, _, tok, pr) in zip(held, sets):
            got = dev.get(tok)
            for r in range(rows):
                t, k, q, m = (float(np.float32(x)) for x in ph[r])
                want, _, near = ref.sample(lh[r].astype(np.float64), t, int(k), q, m, float(uh[r]))
                assert near > 1e-10 and got[r] == want, (turn, r)
    for g in graphs:
        vsl.check(H.vsl_graph_destroy(g))
    vsl.check(H.vsl_stream_destroy(s))
