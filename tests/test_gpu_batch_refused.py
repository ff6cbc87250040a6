"""A step whose requests do not all get their pages: tables, rows into pages, attention. The first new tokens of a request that
was refused belong on a page that it has, where an earlier owner's tokens still lie: no row of it may give an answer over
them. Against 64-bit softmax attention of the requests that were served."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from accelep_amd import capi
from accelep_amd.capi import Batch, CachePaged, check, lib
from batch_helpers import TYPES, dev, ints, pool_of, want_batch
from long_context_helpers import assert_within

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, PAGE = 4, 2, 64, 16


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


class Server:
    """Requests over one cache, and what they hold on the host. Every token that was ever in a page is finite."""

    def __init__(self, rng, requests, pages, width, rows, kind, longest=0):
        self.rng, self.requests, self.rows, self.kind, self.pages = rng, requests, rows, kind, pages
        self.d = {n: ints(x) for n, x in {"lengths": [0] * requests, "seen": [0] * requests, "starts": [0] * (requests + 1),
                                          "table": np.full((requests, width), -1), "slots": [0] * rows, "positions": [0] * rows}.items()}
        self.pool, self.held = pool_of(rng.permutation(pages), pages, PAGE)
        self.planes = [dev(np.full((pages, PAGE, KV, DIM), 0.5, TYPES[kind])) for _ in "kv"]
        b = {n: x.buffer for n, x in self.d.items()}
        self.cache = CachePaged(self.planes[0].buffer, self.planes[1].buffer, capi.CACHE_F16 if kind == "f16" else capi.CACHE_F32,
                                pages, PAGE, KV, DIM)
        self.batch = Batch(b["seen"], b["starts"], b["table"], requests, rows, width, longest, b["slots"])
        self.past = [[np.zeros((0, KV, DIM), TYPES[kind]) for _ in "kv"] for _ in range(requests)]

    def new_tokens(self):
        self.q = self.rng.standard_normal((self.rows, HEADS, DIM)).astype(np.float32)
        self.kv = [self.rng.standard_normal((self.rows, KV, DIM)).astype(np.float32) for _ in "kv"]
        self.on_device = [dev(x) for x in (self.q, *self.kv)]
        self.out = dev(np.full((self.rows, HEADS, DIM), 3.0, np.float32))

    def calls(self, counts, window=0):
        q, k, v = (x.buffer for x in self.on_device)
        b, L = {n: x.buffer for n, x in self.d.items()}, lib()
        check(L.accel_hip_batch_tables(counts.buffer, b["lengths"], C.byref(self.pool), C.byref(self.batch), b["slots"], b["positions"],
                                       b["lengths"], self.held[1].buffer))
        check(L.accel_hip_append_paged(k, v, C.byref(self.cache), b["slots"], self.rows, 0))
        check(L.accel_hip_attention_paged(q, C.byref(self.cache), C.byref(self.batch), self.out.buffer, HEADS, 0, window))

    def step(self, counts, refused, window=0, run=None):
        self.new_tokens()
        cd = ints(counts)
        (run or self.calls)(cd, window)
        got, at = self.out.numpy(), 0
        assert self.held[1].numpy()[1] == len(refused)
        for r, n in enumerate(counts):
            mine = slice(at, at + n)
            at += n
            if r in refused:
                assert n > 0 and np.isnan(got[mine]).all(), f"request {r} was refused and got an answer"
                continue
            seen = len(self.past[r][0])
            self.past[r] = [np.concatenate([p, x[mine].astype(TYPES[self.kind])]) for p, x in zip(self.past[r], self.kv)]
            if n:
                rows = np.unique(np.r_[0:n:13, n - 1])
                rows, want, bound = want_batch(self.q[mine], [self.past[r][0]], [self.past[r][1]], [seen], [0, n], window, rows)
                assert_within(got[mine][rows], want, bound)
        assert (got[at:] == 3.0).all(), "padding rows were written"
        assert self.d["lengths"].numpy().tolist() == [len(p[0]) for p in self.past]

    def release(self, keep):
        kd = ints(keep)
        check(lib().accel_hip_release_pages(kd.buffer, self.d["lengths"].buffer, C.byref(self.pool), C.byref(self.batch)))
        self.past = [[x[:k] for x in p] for p, k in zip(self.past, keep)]


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("longest", [False, True])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("length,new", [(10, 7), (10, 20), (10, 150), (15, 2), (2010, 7), (4010, 100)])
def test_a_refused_request_over_pages_that_were_another_s(kind, longest, window, length, new):
    """With few rows and with many, over whole key ranges and divided ones. Then it gets its pages after all."""
    rng = np.random.default_rng(length + new)
    need = -(-length // PAGE)
    x = Server(rng, 3, need + 5, need + 12, max(length, 40) + 200, kind, 0)
    x.step([0, 0, (need + 5) * PAGE], [])  # all pages have had an owner
    x.release([0, 0, 0])
    x.step([length, 40, 5], [])
    count = new if new + length > (need + 1) * PAGE else new + PAGE  # more than the one page that is left
    x.batch.longest = max(count, 3) if longest else 0
    for _ in range(2):
        before = [p.numpy() for p in x.planes]
        x.step([count, 1, 3], [0], window)
        page = x.d["table"].numpy()[0, need - 1]
        for plane, was in zip(x.planes, before):
            np.testing.assert_array_equal(plane.numpy()[page, length % PAGE or PAGE:], was[page, length % PAGE or PAGE:])
    x.release([length, 0, len(x.past[2][0])])
    x.step([min(count, 3 * PAGE), 0, 1], [], window)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("new", [7, 60])
def test_a_request_that_its_table_row_is_too_short_for(kind, new):
    """Its last page has room for some of the new tokens, its row of the table for no further page."""
    rng = np.random.default_rng(new)
    x = Server(rng, 2, 12, 3, 300, kind)
    x.step([3 * PAGE, 3 * PAGE], [])
    x.release([0, 0])
    x.step([2 * PAGE + 10, 5], [])
    x.step([new, 2], [0])
    x.step([6, 2], [])


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_refused_in_a_graph_that_is_replayed(kind):
    """The same captured step refuses a request, serves it once there are pages, and refuses it again."""
    rng = np.random.default_rng(51)
    x = Server(rng, 3, 6, 8, 120, kind)
    x.step([0, 0, 6 * PAGE], [])
    x.release([0, 0, 0])
    x.new_tokens()
    cd, graph, L = ints([0, 0, 0]), C.c_void_p(), lib()
    held = x.on_device, x.out
    check(L.accel_hip_capture_begin())
    x.calls(cd)
    check(L.accel_hip_capture_end(C.byref(graph)))

    def replay(counts, window):
        for to, fresh in zip([*held[0], held[1]], [*x.on_device, x.out]):
            to.upload(fresh.numpy())
        x.on_device, x.out = held
        cd.upload(counts.numpy())
        check(L.accel_hip_graph_launch(graph, 1))

    try:
        x.step([10, 40, 20], [], run=replay)
        x.step([20, 1, 1], [0], run=replay)
        x.step([20, 1, 1], [0], run=replay)
        x.release([10, 0, 22])
        x.step([20, 0, 1], [], run=replay)
        x.step([60, 17, 1], [0, 1], run=replay)
    finally:
        check(L.accel_hip_graph_destroy(graph))
