"""Captured graphs replayed while other threads use the same stream: a replay is one operation there, so graphs that share a
workspace, and calls that write to it, give what they give in turn, in any order."""
import ctypes
import threading

import numpy as np
import pytest

import vsl_testlib

pytestmark = pytest.mark.gpu
D, REPLAYS = 256, 1500


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


class Chains:
    """Graphs of n kernels each: a number copied from workspace to workspace, which all of them share, and added to the
    graph's own sum by its last kernel (multiples of small integers, exact in fp32)."""

    def __init__(self, vsl, H, dev, kernels, numbers):
        p, self.vsl, self.H, self.dev, self.numbers = dev.p, vsl, H, dev, numbers
        eye = dev.put(np.eye(D, dtype=np.float16))
        self.work = [dev.empty((D,), np.float32) for _ in range(max(kernels))]
        self.sums = [dev.empty((D,), np.float32) for _ in kernels]
        self.stream, self.graphs = ctypes.c_void_p(), []
        starts = [dev.put(np.full(D, v, np.float32)) for v in numbers]
        dev.sync()
        vsl.check(H.vsl_stream_create(ctypes.byref(self.stream)))
        for n, at, total in zip(kernels, starts, self.sums):
            g, s = ctypes.c_void_p(), self.stream
            vsl.check(H.vsl_graph_begin(s))
            for w in self.work[:n - 1]:
                vsl.check(H.vsl_norm_gemv(p(at), None, 1e-5, p(eye), vsl.VSL_DT_F16, D, D, p(w), None, s))
                at = w
            vsl.check(H.vsl_gemv_residual(p(eye), vsl.VSL_DT_F16, D, D, p(at), p(total), None, s))
            vsl.check(H.vsl_graph_end(s, ctypes.byref(g)))
            self.graphs.append(g)

    def run(self, calls):
        """Each call REPLAYS times in a thread of its own, all at once; then every graph's sum is right."""
        ready, codes = threading.Barrier(len(calls)), []

        def go(call):
            ready.wait()
            codes.append({call() for _ in range(REPLAYS)})

        threads = [threading.Thread(target=go, args=(c,)) for c in calls]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        self.dev.sync()
        assert codes == [{0}] * len(calls)
        for v, total in zip(self.numbers, self.sums):
            assert np.array_equal(self.dev.get(total), np.full(D, v * REPLAYS, np.float32))
        for g in self.graphs:
            self.vsl.check(self.H.vsl_graph_destroy(g))
        self.vsl.check(self.H.vsl_stream_destroy(self.stream))


@pytest.mark.parametrize("default_stream", [False, True])
@pytest.mark.parametrize("kernels", [(2, 2), (3, 3), (4, 4), (1, 4), (2, 7), (4, 6), (6, 6), (2, 3, 4, 5)], ids=str)
def test_replays_do_not_mix(vsl, dev, H, kernels, default_stream):
    c = Chains(vsl, H, dev, kernels, [1.0, 512.0, 3.0, 1024.0][:len(kernels)])
    s = None if default_stream else c.stream
    c.run([lambda g=g: H.vsl_graph_launch(g, s) for g in c.graphs])


@pytest.mark.parametrize("n", [2, 3, 4, 6])
def test_calls_do_not_come_between(vsl, dev, H, n):
    """Another thread's own launches on the stream write to the graph's workspace: every replay copies its number there
    anew before it is read, if nothing comes between."""
    c = Chains(vsl, H, dev, (n,), [1.0])
    c.run([lambda: H.vsl_graph_launch(c.graphs[0], c.stream),
           lambda: H.vsl_fill_const(dev.p(c.work[(n - 1) // 2 if n > 2 else 0]), vsl.VSL_DT_F32, D, 512.0, c.stream)])
