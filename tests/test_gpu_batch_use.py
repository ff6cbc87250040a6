"""Batches of requests over a cache in pages as a program uses them: from threads, in graphs that share workspaces, with
pages shared or given up, in caches past 32-bit offsets, in many requests of all lengths. Against 64-bit softmax
attention of each request by itself."""

from __future__ import annotations

import ctypes as C
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest

from accelep_amd import capi
from accelep_amd.capi import Batch, CachePaged, check, lib
from accelep_amd.device import DeviceArray
from batch_helpers import Paged, dev, ints, packed_call, pool_of, tables, want_batch
from long_context_helpers import assert_within

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16"]


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


def compare(x, got, window=0, rows=None):
    at, want, bound = x.want(window, rows)
    assert_within(got[at], want, bound)
    assert (got[sum(x.new):] == 3.0).all(), "padding rows were written"


def some_rows(rng, x, each=4):
    """Of every request the first row, the last and some between."""
    return np.unique(np.concatenate([np.r_[s, s + n - 1, s + rng.integers(0, n, each)] for s, n in zip(x.starts, x.new) if n]))


# Head dims between the kernels' own, tiles of many rows and of few, groups past a tile's rows.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 65), (4, 2, 72), (2, 1, 81), (6, 3, 90), (4, 4, 96), (2, 2, 97), (4, 2, 192),
                                                (40, 2, 64), (130, 1, 32), (2, 2, 8), (2, 2, 4)])
def test_head_dims_and_groups(kind, heads, kv_heads, dim):
    rng = np.random.default_rng(dim + heads)
    x = Paged(rng, [250, 31, 7], [45, 1, 130], 16, heads, kv_heads, dim, kind, pad=2)
    compare(x, x.call(), rows=some_rows(rng, x))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [0, 300])
def test_prompts_of_all_lengths_beside_hundreds_of_steps(kind, window):
    """More requests than a workgroup has threads, long tiles and short ones among those past it."""
    rng = np.random.default_rng(31 + window)
    new = rng.choice([0, 1, 1, 1, 2, 9, 40], 530)
    seen = rng.integers(0, 60, 530)
    for r, s, n in ((3, 0, 700), (255, 2000, 150), (256, 1500, 1), (257, 10, 400), (400, 0, 129), (529, 3000, 300)):
        seen[r], new[r] = s, n
    x = Paged(rng, seen.tolist(), new.tolist(), 32, 4, 2, 64, kind, pad=3)
    rows = np.unique(np.concatenate([rng.integers(0, sum(x.new), 100),
                                     *[x.starts[r] + rng.integers(0, max(new[r], 1), 12) for r in (3, 255, 256, 257, 400, 529)]]))
    compare(x, x.call(window), window, rows)


def test_hundreds_of_packed_prompts():
    rng = np.random.default_rng(32)
    lengths = rng.integers(0, 30, 300)
    lengths[[7, 270, 299]] = 900, 1500, 260
    starts = np.concatenate([[0], np.cumsum(lengths)])
    n = int(starts[-1])
    q, k, v = (rng.standard_normal((n, h, 64)).astype(np.float32) for h in (3, 1, 1))
    parts = [[x[a:b] for a, b in zip(starts, starts[1:])] for x in (k, v)]
    rows = np.unique(np.concatenate([rng.integers(0, n, 150), *[starts[r] + rng.integers(0, lengths[r], 20) for r in (7, 270, 299)]]))
    at, want, bound = want_batch(q, *parts, [0] * 300, starts, 0, rows)
    assert_within(packed_call(q, k, v, starts, 3, 1, 64, n)[at], want, bound)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 150]])
def test_pages_before_the_window_may_be_given_up(kind, new):
    rng = np.random.default_rng(33)
    window, page = 100, 16
    x = Paged(rng, [900, 100, 2500], new, page, 4, 2, 64, kind)
    whole = x.call(window)
    for r, seen in enumerate(x.seen):
        x.table[r, :max(0, seen - window + 1) // page] = -1
    x.upload()
    got = x.call(window)
    np.testing.assert_array_equal(got, whole)
    compare(x, got, window, some_rows(rng, x))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 50])
def test_requests_may_share_the_pages_of_a_prefix(kind, new):
    rng = np.random.default_rng(34)
    x = Paged(rng, [200, 300, 64], [new, 1, new], 16, 4, 2, 64, kind)
    for r, tokens in ((1, 192), (2, 64)):
        x.table[r, :tokens // 16] = x.table[0, :tokens // 16]
        for one in (x.k, x.v):
            one[r] = one[r].copy()
            one[r][:tokens] = one[0][:tokens]
    x.upload()
    compare(x, x.call())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 70])
def test_a_cache_past_32_bit_offsets(kind, new):
    """2^32 elements and some in each plane: rows go into the last pages and are read from there."""
    rng = np.random.default_rng(35)
    kv, dim, page, heads, tokens = 32, 128, 256, 32, 300 + new
    pages = (1 << 32) // (kv * dim * page) + 4
    planes = [DeviceArray((pages * page, kv, dim), np.float16 if kind == "f16" else np.float32) for _ in "kv"]
    cache = CachePaged(planes[0].buffer, planes[1].buffer, capi.CACHE_F16 if kind == "f16" else capi.CACHE_F32, pages, page, kv, dim)
    table = np.array([[pages - 1, 0]], np.int32)
    slots = np.array([table[0, t // page] * page + t % page for t in range(tokens)], np.int32)
    # Nothing else of the planes is read but rows of the same pages past the last token, whose values have no say.
    k, v = (rng.standard_normal((tokens, kv, dim)).astype(np.float32) for _ in "kv")
    kd, vd, sd = dev(k), dev(v), ints(slots)
    L = lib()
    check(L.accel_hip_append_paged(kd.buffer, vd.buffer, C.byref(cache), sd.buffer, tokens, 0))
    q = rng.standard_normal((new, heads, dim)).astype(np.float32)
    held = [ints(a) for a in ([tokens - new], [0, new], table)]
    batch = Batch(*[h.buffer for h in held], 1, new, 2, new)
    qd, out = dev(q), dev(np.zeros_like(q))
    check(L.accel_hip_attention_paged(qd.buffer, C.byref(cache), C.byref(batch), out.buffer, heads, 0, 0))
    rounded = [a.astype(np.float16 if kind == "f16" else np.float32) for a in (k, v)]
    at, want, bound = want_batch(q, [rounded[0]], [rounded[1]], [tokens - new], [0, new], 0, np.unique([0, new // 2, new - 1]))
    assert_within(out.numpy()[at], want, bound)
    for p in planes:
        p.free()


@pytest.mark.parametrize("kind", KINDS)
def test_starts_that_descend(kind):
    """Rows of two requests at once: nothing outside the call's own memory is written, and the next call is right."""
    rng = np.random.default_rng(36)
    x = Paged(rng, [4000, 30, 4000, 700], [200, 1, 200, 100], 16, 4, 2, 64, kind, pad=2)
    good = x.call()
    n = x.rows - 2
    for starts in ([0, n, 0, n, 0], [n, 0, n, 0, n], [0, n, 5, 6, n]):
        x.d["starts"].upload(np.array(starts, np.int32))
        assert (x.call()[n:] == 3.0).all()
    x.d["starts"].upload(x.starts)
    np.testing.assert_array_equal(x.call(), good)


@pytest.mark.parametrize("name", "kv")
@pytest.mark.parametrize("tokens", [[0], [70], [290], [0, 290], [33, 34, 130, 131, 200]])
@pytest.mark.parametrize("power", [-30, -12, 12, 30])
def test_few_rows_of_another_magnitude(name, tokens, power):
    """Tiles of rows of ordinary size before, between and behind tiles that hold one of another, in prompts' tiles."""
    rng = np.random.default_rng(power + 100 + tokens[-1])

    def make(which, r, total):
        x = rng.standard_normal((total, 2, 64))
        if which == name:
            x[tokens] *= 2.0 ** (power if name == "v" else min(power, 4))
        return x

    x = Paged(rng, [260], [60], 16, 8, 2, 64, "f32", make=make)
    at, want, bound = x.want()
    # What a weight or value loses of its 22 bits, at most 2^-24 of the largest value that a row sees, for each key.
    big = max(np.abs(v.astype(np.float64)).max() for v in x.v)
    assert_within(x.call()[at], want, bound + 2.0 ** -24 * 320 * big * 2.0 ** -3)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("order", [1, -1])
def test_scores_that_grow_or_fall_along_the_keys(kind, order):
    """The largest score of a row moves with nearly every tile, or is the first tile's."""
    rng = np.random.default_rng(43)

    def make(which, r, total):
        x = rng.standard_normal((total, 2, 64))
        return x * (np.linspace(0.05, 12, total)[::order, None, None] if which == "k" else 1)

    x = Paged(rng, [300, 700], [50, 1], 16, 8, 2, 64, kind, make=make)
    compare(x, x.call())


# ---- threads and graphs --------------------------------------------------------------------------

def attention_job(rng, kind, seen, new, window=0):
    x = Paged(rng, seen, new, 16, 8, 2, 64, kind)
    qd = dev(x.q)

    def call(out):
        check(lib().accel_hip_attention_paged(qd.buffer, C.byref(x.cache), C.byref(x.batch), out.buffer, 8, 0, window))

    return call, lambda: dev(np.zeros((x.rows, 8, 64), np.float32)), (x, qd)


def tables_job(rng, requests=2500):
    """More requests than one workgroup describes: two launches, what is between them in the attention's workspace."""
    counts, lengths, page = rng.integers(0, 4, requests), rng.integers(0, 50, requests), 16
    rows, width = int(counts.sum()) + 3, 5
    stack = rng.permutation(requests).astype(np.int32)
    old = np.full((requests, width), -1, np.int32)
    for r, n in enumerate(lengths):
        old[r, :-(-int(n) // page)] = 7
    want = tables(counts, lengths, old, stack, requests, rows, page, requests)
    pool, held = pool_of(stack, requests, page)
    cd, ld = ints(counts), ints(lengths)
    keep = [pool, held, cd, ld]

    def call(out):
        d = out.d
        batch = Batch(d["seen"].buffer, d["starts"].buffer, d["table"].buffer, requests, rows, width, 0)
        check(lib().accel_hip_batch_tables(cd.buffer, ld.buffer, C.byref(pool), C.byref(batch), d["slots"].buffer,
                                           d["positions"].buffer, d["after"].buffer, d["state"].buffer))

    class Out:
        def __init__(self):
            self.d = {"seen": ints([0] * requests), "starts": ints([0] * (requests + 1)), "table": ints(old),
                      "slots": ints([0] * rows), "positions": ints([0] * rows), "after": ints([0] * requests), "state": ints([0, 0])}

        def numpy(self):
            return np.concatenate([self.d[n].numpy().ravel() for n in ("starts", "slots", "positions", "after", "state", "table")])

    flat = np.concatenate([np.asarray(want[n]).ravel() for n in ("starts", "slots", "positions", "lengths_after", "state_after", "table")])
    return call, Out, (keep, flat)


def test_calls_from_two_threads():
    """Attention that divides key ranges, and tables in two launches, share a workspace: the threads' launches meet on
    the one stream."""
    rng = np.random.default_rng(37)
    jobs = [[attention_job(rng, "f32", [5000, 30], [1, 1]), attention_job(rng, "f16", [2500, 900, 3], [100, 1, 40])],
            [tables_job(rng), attention_job(rng, "f32", [1500, 900], [60, 1])]]
    wants = []
    for job in jobs:
        wants.append([])
        for call, make, _ in job:
            out = make()
            call(out)
            wants[-1].append(out.numpy())
    np.testing.assert_array_equal(wants[1][0], jobs[1][0][2][1])
    outs = [[[make() for _, make, _ in job] for _ in range(25)] for job in jobs]
    failures = []

    def run(job, mine):
        try:
            for each in mine:
                for (call, _, _), out in zip(job, each):
                    call(out)
        except BaseException as e:  # handed to the test's thread
            failures.append(e)

    threads = [threading.Thread(target=run, args=a) for a in zip(jobs, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    for mine, want in zip(outs, wants):
        for each in mine:
            for out, w in zip(each, want):
                np.testing.assert_array_equal(out.numpy(), w)


def test_two_graphs_that_share_a_workspace():
    """Replayed in turn, with the same calls and other calls eagerly between."""
    rng = np.random.default_rng(38)
    jobs = [attention_job(rng, "f32", [5000, 30], [1, 1]), attention_job(rng, "f16", [2500, 900, 3], [100, 1, 40]), tables_job(rng)]
    between = attention_job(rng, "f32", [8000], [3])
    L = lib()
    outs, wants, graphs = [], [], []
    for call, make, _ in [*jobs, between]:
        out = make()
        call(out)
        outs.append(out)
        wants.append(out.numpy())
    for (call, _, _), out in zip(jobs, outs):
        check(L.accel_hip_capture_begin())
        call(out)
        graph = C.c_void_p()
        check(L.accel_hip_capture_end(C.byref(graph)))
        graphs.append(graph)
    try:
        for times in (1, 2, 1, 3):
            for graph, out, want in zip(graphs, outs, wants):
                if isinstance(out, DeviceArray):
                    out.upload(np.full(out.shape, -1.0, np.float32))
                else:
                    out.d["slots"].upload(np.full(out.d["slots"].shape, -5, np.int32))
                check(L.accel_hip_graph_launch(graph, times))
                between[0](outs[-1])
                np.testing.assert_array_equal(out.numpy(), want)
                np.testing.assert_array_equal(outs[-1].numpy(), wants[-1])
    finally:
        for graph in graphs:
            check(L.accel_hip_graph_destroy(graph))


FIRST_IN_A_CAPTURE = """
import ctypes as C, sys
sys.path[:0] = sys.argv[1:]
import numpy as np
from accelep_amd.capi import check, lib
from batch_helpers import Paged, dev
from long_context_helpers import assert_within
from test_gpu_batch_use import tables_job
L = lib()
check(L.accel_hip_init())
r = np.random.default_rng(39)
call, make, _ = tables_job(r)
out, graph = make(), C.c_void_p()
check(L.accel_hip_capture_begin())
try:
    call(out)
    print("no refusal", flush=True)
except Exception as e:
    print("refused" if "temporary buffer" in str(e) else repr(e), flush=True)
check(L.accel_hip_capture_end(C.byref(graph)))
check(L.accel_hip_graph_destroy(graph))
for kind, new in (("f32", [1, 1]), ("f16", [130, 1])):
    x = Paged(r, [3000, 40], new, 16, 4, 2, 64, kind)
    q, out = dev(x.q), dev(np.zeros((x.rows, 4, 64), np.float32))
    graph = C.c_void_p()
    check(L.accel_hip_capture_begin())
    check(L.accel_hip_attention_paged(q.buffer, C.byref(x.cache), C.byref(x.batch), out.buffer, 4, 0, 0))
    check(L.accel_hip_capture_end(C.byref(graph)))
    rows = np.unique(np.linspace(0, x.rows - 1, 9).astype(int))
    at, want, bound = x.want(rows=rows)
    for replay in range(3):
        out.upload(np.full(out.shape, -1.0, np.float32))
        check(L.accel_hip_graph_launch(graph, 1))
        assert_within(out.numpy()[at], want, bound)
    check(L.accel_hip_graph_destroy(graph))
    assert_within(x.call()[at], want, bound)
    print("held", flush=True)
"""


def test_a_first_call_inside_a_capture():
    """Before any eager call there is no workspace: key ranges stay whole, tables that need one are refused."""
    here = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE, str(here), str(here.parent)], capture_output=True, text=True,
                       timeout=100)
    assert r.returncode == 0 and r.stdout.split() == ["refused", "held", "held"], r.stdout + r.stderr


def test_the_live_allocations_do_not_change():
    L = lib()
    rng = np.random.default_rng(40)
    jobs = [attention_job(rng, "f32", [500, 30], [1, 60]), tables_job(rng)]
    outs = [make() for _, make, _ in jobs]
    for (call, _, _), out in zip(jobs, outs):
        call(out)
    live = L.accel_hip_live_allocs()
    for (call, _, _), out in zip(jobs, outs):
        for _ in range(3):
            call(out)
    assert L.accel_hip_live_allocs() == live
