"""Scaled tables, partial rotation, attention with modified scores and sampling of rows, run together as a model's steps
run them: prompts in several calls, tokens by a captured graph, several sequences on streams of their own.

Each stage is checked against its 64-bit definition from what the stage before left on the device, with the tolerances of the
operators' own tests (u = 2^-24): rotation 3 u (|a| + |b|) and the output's rounding; attention key by key as
token_step_ref.attention bounds it; a logit's sum of K products K u of their magnitudes; tokens equal but within 1e-10 of a
border."""
import ctypes
import math

import numpy as np
import pytest

import token_step_ref as ref
import vsl_testlib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
N_Q, N_KV, HD, ROT, V = 8, 2, 128, 64, 5000
CAP, TABLE, SCALE, SOFTCAP, NSPLIT = 400, 500, 0.09, 30.0, 8
SAMPLERS = [(0.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.2, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.9, 300, 0.9, 0.01)]


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


class Model:
    """A layer's weights that a step needs: tables, slopes and an output matrix."""

    def __init__(self, vsl, H, dev, rng):
        self.vsl, self.H, self.dev = vsl, H, dev
        scaling = vsl.RopeScaling(type=3, theta=1e4, factor=8.0, orig_ctx=64.0, low=1.0, high=8.0)
        self.cos, self.sin = dev.empty((TABLE, ROT // 2), np.float32), dev.empty((TABLE, ROT // 2), np.float32)
        vsl.check(H.vsl_rope_tables(ROT, 0, TABLE, ctypes.byref(scaling), None, dev.p(self.cos), dev.p(self.sin), None))
        a = np.arange(TABLE)[:, None] * ref.rope_freqs(ROT, 1e4, 3, 8.0, 64.0, 1.0, 8.0)
        m = 0.1 * math.log(8.0) + 1
        self.c, self.s = np.cos(a) * m, np.sin(a) * m
        assert np.all(np.abs(dev.get(self.cos) - self.c) <= (U + 2.0 ** -29) * m * 1.01)
        self.slopes_host = (2.0 ** -np.arange(1, N_Q + 1)).astype(np.float32)
        self.slopes = dev.put(self.slopes_host)
        self.W = (rng.normal(0, 0.2, (V, N_Q * HD))).astype(np.float16)
        self.Wd = dev.put(self.W)


class Sequence:
    """Caches, buffers and workspaces of one sequence, and its calls."""

    def __init__(self, m, rows):
        dev = m.dev
        self.m, self.rows = m, rows
        self.kc, self.vc = (dev.put(np.full((N_KV, CAP, HD), np.nan, np.float16)) for _ in range(2))
        self.qkv = dev.empty((rows, N_Q + 2 * N_KV, HD), np.float32)
        self.q, self.out = dev.empty((2, rows, N_Q, HD), np.float16), dev.empty((2, rows, N_Q, HD), np.float16)
        self.at, self.ranges = dev.empty((rows,), np.uint32), dev.empty((rows, 2), np.uint32)
        self.n = max(m.H.vsl_attn_prefill_mods_ws_bytes(rows, p, N_Q, N_KV, HD) for p in range(0, CAP - rows + 1, 10))
        self.ws = dev.empty((max(self.n, 16),), np.uint8)
        self.row, self.q1, self.o1 = dev.empty((N_Q + 2 * N_KV, HD), np.float32), *(dev.empty((N_Q, HD), np.float32) for _ in range(2))
        self.place, self.window = dev.empty((1,), np.uint32), dev.empty((1, 2), np.uint32)
        self.po, self.pml = dev.empty((N_Q, NSPLIT, HD), np.float32), dev.empty((N_Q, NSPLIT, 2), np.float32)
        self.ctrl, self.logits = dev.empty((8,), np.uint32), dev.empty((1, V), np.float32)
        self.params, self.u = dev.empty((1, 4), np.float32), dev.empty((1,), np.float32)
        self.n_rows = m.H.vsl_sample_rows_ws_bytes(1, V)
        self.ws_rows = dev.empty((self.n_rows,), np.uint8)
        self.token, self.share = dev.empty((1,), np.uint32), dev.empty((1,), np.float32)

    def prompt(self, S, pos0, stream=None):
        m, p = self.m, self.m.dev.p
        m.vsl.check(m.H.vsl_rope_part_append(p(self.qkv), S, N_Q, N_KV, HD, ROT, 1, pos0, p(self.at), p(m.cos), p(m.sin), TABLE,
                                             p(self.q), 2, p(self.kc), p(self.vc), 1, CAP, stream))
        mods = m.vsl.AttnMods(softcap=SOFTCAP, slopes=p(m.slopes), ranges=p(self.ranges))
        m.vsl.check(m.H.vsl_attn_prefill_mods(p(self.q), 2, p(self.kc), p(self.vc), S, pos0, N_Q, N_KV, HD, CAP, SCALE, p(self.out), 2,
                                              ctypes.byref(mods), p(self.ws), self.n, stream))

    def step(self, stream=None):
        m, p = self.m, self.m.dev.p
        m.vsl.check(m.H.vsl_rope_part_append_decode(p(self.row), N_Q, N_KV, HD, ROT, 1, p(self.place), p(m.cos), p(m.sin), TABLE,
                                                    p(self.q1), p(self.kc), p(self.vc), 1, CAP, p(self.ctrl), stream))
        mods = m.vsl.AttnMods(softcap=SOFTCAP, slopes=p(m.slopes), ranges=p(self.window))
        m.vsl.check(m.H.vsl_attn_decode_mods(p(self.q1), p(self.kc), p(self.vc), 1, N_Q, N_KV, HD, CAP, SCALE, NSPLIT, p(self.po),
                                             p(self.pml), p(self.o1), p(self.ctrl), ctypes.byref(mods), stream))
        m.vsl.check(m.H.vsl_gemv(p(m.Wd), 1, V, N_Q * HD, p(self.o1), 0, 1, p(self.logits), 0, stream))
        m.vsl.check(m.H.vsl_sample_rows(p(self.logits), 0, 1, V, V, p(self.params), p(self.u), p(self.token), p(self.share),
                                        p(self.ws_rows), self.n_rows, stream))

    def fill(self, t, a):
        a = np.ascontiguousarray(a)
        t.view(-1)[:a.size].copy_(self.m.dev.torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).view(-1))

    def set_prompt(self, qkv, at, ranges):
        self.fill(self.qkv, qkv)
        self.fill(self.at, at)
        self.fill(self.ranges, ranges)

    def set_step(self, row, place, window, pos, params, u):
        self.fill(self.row, row)
        self.fill(self.place, np.array([place], np.uint32))
        self.fill(self.window, np.array(window, np.uint32))
        self.fill(self.ctrl, np.array([pos, 0, 0, 0, 9, 0, CAP, 0], np.uint32))
        p = np.array([[params[0], 0, params[2], params[3]]], np.float32)
        p[0, 1:2].view(np.uint32)[0] = params[1]
        self.fill(self.params, p)
        self.fill(self.u, np.array([u], np.float32))

    def check_rotation(self, qkv, at, pos0, got_q, q_err):
        """Queries and the appended keys of a call; returns the caches' rows as 64-bit values."""
        S, dev = qkv.shape[0], self.m.dev
        want, pair = ref.rotate(qkv[:, :N_Q + N_KV], self.m.c[at][:, None], self.m.s[at][:, None], ROT, True)
        tab = (U + 2.0 ** -29) * 1.3 * pair  # the tables' own rounding, mscale below 1.3
        assert np.all(np.abs(got_q - want[:, :N_Q]) <= (3 * U * 1.3 * pair + tab)[:, :N_Q] + q_err(np.abs(want[:, :N_Q])))
        K, Vv = (dev.get(c).astype(np.float64)[:, :pos0 + S] for c in (self.kc, self.vc))
        k = want[:, N_Q:].transpose(1, 0, 2)
        tol = (3 * U * 1.3 * pair + tab)[:, N_Q:].transpose(1, 0, 2)
        assert np.all(np.abs(K[:, pos0:] - k) <= tol + np.maximum(2.0 ** -11 * np.abs(k), 2.0 ** -25) * 1.001)
        assert np.array_equal(Vv[:, pos0:], qkv[:, N_Q + N_KV:].transpose(1, 0, 2).astype(np.float16).astype(np.float64))
        return K, Vv

    def check_prompt(self, qkv, at, ranges, pos0):
        S, dev = qkv.shape[0], self.m.dev
        two = lambda t: dev.get(t).reshape(2, -1)[:, :S * N_Q * HD].astype(np.float64).sum(0).reshape(S, N_Q, HD)
        got_q, got = (two(t) for t in self.planes(S))
        K, Vv = self.check_rotation(qkv, at, pos0, got_q, lambda a: 2.0 ** -22 * a + 2.0 ** -25)
        want, err = ref.attention(got_q, K, Vv, float(np.float32(SCALE)), pos0 + np.arange(S), SOFTCAP, self.m.slopes_host, ranges,
                                  2 * HD * U + 6 * U, 2.0 ** -21)
        a = np.abs(want)
        assert np.all(np.abs(got - want) <= (err + 2.0 ** -22 * a + 2.0 ** -25) * 1.001 + 2 * U * a)

    def planes(self, S):
        """q and out of a call of S rows: both planes lie S rows apart."""
        n = S * N_Q * HD
        return [t.view(-1)[:2 * n] for t in (self.q, self.out)]

    def check_step(self, row, place, window, pos, params, u):
        dev = self.m.dev
        q = dev.get(self.q1).astype(np.float64)
        K, Vv = self.check_rotation(row[None], np.array([place]), pos, q[None], lambda a: U * a)
        want, err = ref.attention(q[None], K, Vv, float(np.float32(SCALE)), [pos], SOFTCAP, self.m.slopes_host, [window],
                                  HD * U + 2.0 ** -21 + 6 * U, 2.0 ** -21)
        o = dev.get(self.o1).astype(np.float64)
        assert np.all(np.abs(o - want[0]) <= err[0] + 2 * U * np.abs(want[0]) + 1e-30)
        W, o, l = self.m.W.astype(np.float64), o.reshape(-1), dev.get(self.logits)[0].astype(np.float64)
        assert np.all(np.abs(l - W @ o) <= N_Q * HD * U * (np.abs(W) @ np.abs(o)) + 1e-30)
        p = [float(np.float32(x)) for x in params]
        tok, share, near = ref.sample(l, p[0], int(p[1]), p[2], p[3], float(np.float32(u)))
        assert near > 1e-10
        assert dev.get(self.token, np.uint32)[0] == tok
        assert abs(float(dev.get(self.share)[0]) - share) <= 2.0 ** -24 * share * 1.001 + 1e-10


def packed(docs, pos0, pad):
    """Positions and ranges of documents of the given lengths, then rows of padding."""
    at, rg, b = [], [], 0
    for n in docs:
        at += list(range(n))
        rg += [(pos0 + b, pos0 + b + i + 1) for i in range(n)]
        b += n
    return np.array(at + [TABLE - 1] * pad, np.uint32), np.array(rg + [(0, 0)] * pad, np.uint32)


def rows(rng, S):
    return rng.normal(0, 1.2, (S, N_Q + 2 * N_KV, HD)).astype(np.float32)


def tokens_of(rng, n, first, pos):
    """Inputs of n tokens that continue a document which began at `first`, the last ones of a window of 50."""
    for i in range(n):
        begin = first if i < n // 2 else max(first, pos + i - 49)
        yield (rows(rng, 1)[0], pos + i - first, (begin, 0xFFFFFFFF), pos + i, SAMPLERS[i % len(SAMPLERS)], float(rng.random()))


def test_prompts_then_tokens(vsl, H, dev):
    """Packed documents and rows of padding, more rows of the last document (appended over the padding), then its tokens:
    eager, and by a graph captured once, with the program's own work between the replays."""
    rng = np.random.default_rng(21)
    m = Model(vsl, H, dev, rng)
    s = Sequence(m, 150)
    x, (at, rg) = rows(rng, 150), packed((1, 40, 33, 70), 0, 6)
    s.set_prompt(x, at, rg)
    s.prompt(150, 0)
    s.check_prompt(x, at, rg, 0)
    assert not np.any(dev.get(s.out)[:, 144:])
    x, at = rows(rng, 45), np.arange(70, 115).astype(np.uint32)  # the last document began at 74
    rg = np.array([(74, 144 + i + 1) for i in range(45)], np.uint32)
    s.set_prompt(x, at, rg)
    s.prompt(45, 144)
    s.check_prompt(x, at, rg, 144)
    graph, st = ctypes.c_void_p(), ctypes.c_void_p()
    for args in tokens_of(rng, 4, 74, 189):
        s.set_step(*args)
        s.step()
        s.check_step(*args)
    vsl.check(H.vsl_stream_create(ctypes.byref(st)))
    dev.torch.cuda.synchronize()
    vsl.check(H.vsl_graph_begin(st))
    s.step(st)
    vsl.check(H.vsl_graph_end(st, ctypes.byref(graph)))
    for args in tokens_of(rng, 12, 74, 193):
        s.set_step(*args)
        dev.torch.ones(1000, device="cuda").sum().item()
        vsl.check(H.vsl_graph_launch(graph, st))
        vsl.check(H.vsl_stream_sync(st))
        s.check_step(*args)
    vsl.check(H.vsl_graph_destroy(graph))
    vsl.check(H.vsl_stream_destroy(st))


def test_sequences_at_once(vsl, H, dev):
    """Three sequences on streams of their own without a wait between, one of them replaying a graph of its prompt: bit for
    bit what each gives alone."""
    rng = np.random.default_rng(22)
    m = Model(vsl, H, dev, rng)
    lengths = (150, 45, 7)
    seqs = [Sequence(m, n) for n in lengths]
    streams, graph = [ctypes.c_void_p() for _ in lengths], ctypes.c_void_p()
    for st in streams:
        vsl.check(H.vsl_stream_create(ctypes.byref(st)))
    for s, n in zip(seqs, lengths):
        s.fill(s.kc, rng.normal(0, 1, (N_KV, CAP, HD)).astype(np.float16))
        s.fill(s.vc, rng.normal(0, 1, (N_KV, CAP, HD)).astype(np.float16))
        at = np.arange(200, 200 + n).astype(np.uint32)
        s.set_prompt(rows(rng, n), at, np.array([(i % 90, 200 + i + 1) for i in range(n)], np.uint32))
        s.set_step(rows(rng, 1)[0], 200 + n, (3, 0xFFFFFFFF), 200 + n, SAMPLERS[n % 5], 0.37)

    def results():
        return [[dev.get(t).copy() for t in (s.q, s.out, s.o1, s.logits, s.token, s.share, s.kc, s.vc)] for s in seqs]

    for s, n in zip(seqs, lengths):
        s.prompt(n, 200)
        s.step()
        dev.torch.cuda.synchronize()
    alone = results()
    assert all(np.all(np.isfinite(a)) for r in alone for a in r) and all(r[2].any() for r in alone)
    vsl.check(H.vsl_graph_begin(streams[1]))
    seqs[1].prompt(lengths[1], 200, streams[1])
    seqs[1].step(streams[1])
    vsl.check(H.vsl_graph_end(streams[1], ctypes.byref(graph)))
    for _ in range(4):
        for s in seqs:
            for t in (s.q, s.out, s.o1, s.logits, s.token, s.share):
                t.fill_(5)
        dev.torch.cuda.synchronize()
        for _ in range(3):
            for i in (0, 2):
                seqs[i].prompt(lengths[i], 200, streams[i])
                seqs[i].step(streams[i])
            vsl.check(H.vsl_graph_launch(graph, streams[1]))
        for st in streams:
            vsl.check(H.vsl_stream_sync(st))
        for a, b in zip(alone, results()):
            assert all(np.array_equal(x, y) for x, y in zip(a, b))
    vsl.check(H.vsl_graph_destroy(graph))
    for st in streams:
        vsl.check(H.vsl_stream_destroy(st))


def test_offsets_past_32_bits(vsl, H, dev):
    """Caches of more than 2^31 values and rows of logits more than 2^32 bytes apart: bit for bit what small ones give."""
    rng = np.random.default_rng(23)
    m = Model(vsl, H, dev, rng)
    S, small, large = 3, 128, 64 * 33000
    assert N_KV * 4 * large * HD > 2 ** 31
    x, at = dev.put(rng.normal(0, 1, (S, N_Q + 8 * N_KV, HD)).astype(np.float32)), dev.put(np.array([7, 8, 9], np.uint32))
    row, place = dev.put(rng.normal(0, 1, (N_Q + 8 * N_KV, HD)).astype(np.float32)), dev.put(np.array([10], np.uint32))
    old = [dev.torch.randn(4 * N_KV, 60, HD, device="cuda").half() for _ in range(2)]
    p, nkv, outs = dev.p, 4 * N_KV, []
    for cap in (small, large):
        kc, vc = (dev.empty((nkv, cap, HD), np.float16) for _ in range(2))
        pos0 = cap - 4
        for c, o in zip((kc, vc), old):
            c[:, pos0 - 60:pos0] = o
        rg = dev.put(np.array([(pos0 - 60, pos0 + 1), (pos0 - 1, pos0 + 2), (0, 0)], np.uint32))
        mods = vsl.AttnMods(softcap=SOFTCAP, slopes=p(m.slopes), ranges=p(rg))
        q, out = dev.empty((2, S, N_Q, HD), np.float16), dev.empty((2, S, N_Q, HD), np.float16)
        vsl.check(H.vsl_rope_part_append(p(x), S, N_Q, nkv, HD, ROT, 1, pos0, p(at), p(m.cos), p(m.sin), TABLE, p(q), 2, p(kc), p(vc),
                                         1, cap, None))
        vsl.check(H.vsl_attn_prefill_mods(p(q), 2, p(kc), p(vc), S, pos0, N_Q, nkv, HD, cap, SCALE, p(out), 2, ctypes.byref(mods),
                                          None, 0, None))
        ctrl, q1, o1 = dev.put(np.array([cap - 1, 0, 0, 0, 9, 0, cap, 0], np.uint32)), *(dev.empty((N_Q, HD), np.float32) for _ in range(2))
        po, pml = dev.empty((N_Q, NSPLIT, HD), np.float32), dev.empty((N_Q, NSPLIT, 2), np.float32)
        vsl.check(H.vsl_rope_part_append_decode(p(row), N_Q, nkv, HD, ROT, 1, p(place), p(m.cos), p(m.sin), TABLE, p(q1), p(kc), p(vc),
                                                1, cap, p(ctrl), None))
        rg1 = dev.put(np.array([(pos0 - 50, 0xFFFFFFFF)], np.uint32))
        mods = vsl.AttnMods(softcap=SOFTCAP, slopes=p(m.slopes), ranges=p(rg1))
        vsl.check(H.vsl_attn_decode_mods(p(q1), p(kc), p(vc), 1, N_Q, nkv, HD, cap, SCALE, NSPLIT, p(po), p(pml), p(o1), p(ctrl),
                                         ctypes.byref(mods), None))
        outs.append([dev.get(t).copy() for t in (q, out, q1, o1, kc[:, pos0 - 60:], vc[:, pos0 - 60:])])
    assert all(np.array_equal(a, b) for a, b in zip(*outs)) and all(a.any() for a in outs[0])
    rows_n, n, stride = len(SAMPLERS), 700, 1 << 28
    logits = rng.normal(0, 2, (rows_n, n)).astype(np.float32)
    far = dev.empty(((rows_n - 1) * stride + n,), np.float32)
    for r in range(rows_n):
        far[r * stride:r * stride + n].copy_(dev.torch.from_numpy(logits[r]))
    par = np.zeros((rows_n, 4), np.float32)
    for r, s in enumerate(SAMPLERS):
        par[r] = (s[0], 0, s[2], s[3])
        par[r, 1:2].view(np.uint32)[0] = s[1]
    u, par = dev.put(rng.random(rows_n).astype(np.float32)), dev.put(par)
    size = H.vsl_sample_rows_ws_bytes(rows_n, n)
    ws, got = dev.empty((size,), np.uint8), []
    for l, st in ((dev.put(logits), n), (far, stride)):
        tok, share = dev.empty((rows_n,), np.uint32), dev.empty((rows_n,), np.float32)
        vsl.check(H.vsl_sample_rows(p(l), 0, rows_n, n, st, p(par), p(u), p(tok), p(share), p(ws), size, None))
        got.append((dev.get(tok), dev.get(share)))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1]) and len(set(got[0][0])) > 1
