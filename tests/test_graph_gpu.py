"""Captured graphs replayed by the C ABI: chains of a few kernels (replayed as launches of their own), longer ones, ones
with a copy in them and ones that fork, each replay compared bit for bit with the same calls made eagerly."""
import ctypes

import numpy as np
import pytest

import vsl_testlib

pytestmark = pytest.mark.gpu
D = 256


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


def stream(vsl, H):
    s = ctypes.c_void_p()
    vsl.check(H.vsl_stream_create(ctypes.byref(s)))
    return s


class Run:
    """A few vectors and a call that adds W times one of them to the next: the order of calls shows in the values."""

    def __init__(self, vsl, H, dev, n, seed):
        rng = np.random.default_rng(seed)
        self.vsl, self.H, self.dev, self.n = vsl, H, dev, n
        self.W = dev.put(rng.normal(0, D ** -0.5, (D, D)).astype(np.float16))
        self.start = rng.normal(0, 1, (n + 1, D)).astype(np.float32)
        self.x = [dev.put(r) for r in self.start]

    def add(self, i, j, s):
        p = self.dev.p
        self.vsl.check(self.H.vsl_gemv_residual(p(self.W), 1, D, D, p(self.x[i]), p(self.x[j]), None, s))

    def copy(self, i, j, s):
        p = self.dev.p
        self.vsl.check(self.H.vsl_copy_d2d(p(self.x[j]), p(self.x[i]), D * 4, s))

    def values(self):
        self.dev.sync()
        return np.stack([self.dev.get(x) for x in self.x])

    def reset(self):
        for x, r in zip(self.x, self.start):
            x.copy_(self.dev.put(r))
        self.dev.sync()


def replays(vsl, H, dev, run, calls, on=None, times=3):
    """The calls eagerly, `times` over, then captured and replayed as often, with eager work between."""
    eager = []
    for _ in range(times):
        calls(None)
        eager.append(run.values())
    run.reset()
    s, g = stream(vsl, H), ctypes.c_void_p()
    vsl.check(H.vsl_graph_begin(s))
    calls(s)
    vsl.check(H.vsl_graph_end(s, ctypes.byref(g)))
    assert np.array_equal(run.values(), run.start)  # a capture runs nothing
    work = [dev.put(np.ones(D, np.float32)) for _ in range(2)]
    for want in eager:
        t = s if on is None else on
        vsl.check(H.vsl_graph_launch(g, t))
        vsl.check(H.vsl_stream_sync(t))
        assert np.array_equal(run.values(), want)
        vsl.check(H.vsl_gemv_residual(dev.p(run.W), 1, D, D, dev.p(work[0]), dev.p(work[1]), None, None))
        dev.sync()
    vsl.check(H.vsl_graph_destroy(g))
    vsl.check(H.vsl_stream_destroy(s))


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 9])
def test_chain(vsl, H, dev, n):
    run = Run(vsl, H, dev, n, 10 + n)
    replays(vsl, H, dev, run, lambda s: [run.add(i, i + 1, s) for i in range(n)])


@pytest.mark.parametrize("n", [3, 6])
def test_chain_on_another_stream(vsl, H, dev, n):
    run = Run(vsl, H, dev, n, 30 + n)
    other = stream(vsl, H)
    replays(vsl, H, dev, run, lambda s: [run.add(i, i + 1, s) for i in range(n)], on=other)
    vsl.check(H.vsl_stream_destroy(other))


def test_a_copy_between_kernels(vsl, H, dev):
    run = Run(vsl, H, dev, 3, 50)

    def calls(s):
        run.add(0, 1, s)
        run.copy(1, 2, s)
        run.add(2, 3, s)
    replays(vsl, H, dev, run, calls)


def test_a_fork(vsl, H, dev):
    run = Run(vsl, H, dev, 4, 60)
    side, fork, join = stream(vsl, H), ctypes.c_void_p(), ctypes.c_void_p()
    for e in (fork, join):
        vsl.check(H.vsl_event_create(ctypes.byref(e)))

    def calls(s):
        run.add(0, 1, s)
        vsl.check(H.vsl_event_record(fork, s))
        vsl.check(H.vsl_stream_wait_event(side, fork))
        run.add(1, 2, side)
        vsl.check(H.vsl_event_record(join, side))
        run.add(1, 3, s)
        vsl.check(H.vsl_stream_wait_event(s, join))
        run.add(2, 4, s)
    replays(vsl, H, dev, run, calls)
    for e in (fork, join):
        vsl.check(H.vsl_event_destroy(e))
    vsl.check(H.vsl_stream_destroy(side))


def test_two_graphs_in_turn(vsl, H, dev):
    """Two chains over the same vectors, replayed in turn on one stream without a wait between."""
    run = Run(vsl, H, dev, 3, 70)
    a = lambda s: [run.add(0, 1, s), run.add(1, 2, s)]
    b = lambda s: [run.add(2, 3, s), run.add(3, 1, s), run.add(1, 0, s)]
    for _ in range(4):
        a(None)
        b(None)
    want = run.values()
    run.reset()
    s, graphs = stream(vsl, H), []
    for calls in (a, b):
        g = ctypes.c_void_p()
        vsl.check(H.vsl_graph_begin(s))
        calls(s)
        vsl.check(H.vsl_graph_end(s, ctypes.byref(g)))
        graphs.append(g)
    for _ in range(4):
        for g in graphs:
            vsl.check(H.vsl_graph_launch(g, s))
    vsl.check(H.vsl_stream_sync(s))
    assert np.array_equal(run.values(), want)
    for g in graphs:
        vsl.check(H.vsl_graph_destroy(g))
    vsl.check(H.vsl_stream_destroy(s))
