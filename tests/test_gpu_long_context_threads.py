"""Attention over divided key ranges from two threads, one of which replays a captured call."""

from __future__ import annotations

import ctypes as C
import threading

import numpy as np
import pytest

from long_context_helpers import Cache, check, dev, lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


def test_a_replayed_graph_and_eager_calls_keep_their_sums_apart():
    """Both write the parts of key ranges to the same memory and join them in a second launch."""
    r = np.random.default_rng(21)
    L = lib()
    calls = []
    for seq, heads, kv, dim, length in ((1, 32, 8, 128, 5000), (3, 9, 3, 64, 9000)):
        cache = Cache(length, kv, dim, 64)
        cache.fill(r, length)
        q = dev(r.standard_normal((seq, heads, dim)).astype(np.float32))
        kf, vf = (dev(cache.values(n)) for n in "kv")

        def call(out, q=q, cache=cache, kf=kf, vf=vf, seq=seq, heads=heads, kv=kv, dim=dim, length=length):
            check(L.accel_hip_attention_q8(q.buffer, C.byref(cache.handle), out[0].buffer, seq, length - seq, heads, 0, 0, 0))
            check(L.accel_hip_attention_window(q.buffer, kf.buffer, vf.buffer, out[1].buffer, seq, length - seq, heads, kv, dim, 0,
                                               4000, 4))

        def outputs(q=q):
            return [dev(np.zeros(q.shape, np.float32)) for _ in range(2)]

        want = outputs()
        call(want)
        calls.append((call, outputs, [w.numpy() for w in want]))
    (captured, new_outputs, graph_want), (eager, new_eager, eager_want) = calls
    captured(new_outputs())  # the workspace has its size
    sets, graphs = [new_outputs() for _ in range(20)], []
    for out in sets:  # a graph for each set of outputs, so that every replay is looked at
        graph = C.c_void_p()
        check(L.accel_hip_capture_begin())
        try:
            captured(out)
        finally:
            check(L.accel_hip_capture_end(C.byref(graph)))
        graphs.append(graph)
    eager_sets = [new_eager() for _ in range(40)]
    failures = []

    def run(work):
        try:
            work()
        except BaseException as e:  # handed to the test's thread
            failures.append(e)

    threads = [threading.Thread(target=run, args=(lambda: [check(L.accel_hip_graph_launch(g, 2)) for g in graphs],)),
               threading.Thread(target=run, args=(lambda: [eager(out) for out in eager_sets],))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    for outs, want in ((sets, graph_want), (eager_sets, eager_want)):
        for out in outs:
            for got, w in zip(out, want):
                np.testing.assert_array_equal(got.numpy(), w)
    for graph in graphs:
        check(L.accel_hip_graph_destroy(graph))
