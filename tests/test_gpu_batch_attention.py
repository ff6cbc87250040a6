"""Attention of a batch of requests, over pages of a cache and over packed prompts, through the C-ABI, against
64-bit softmax attention of each request by itself (long_context_helpers.attend, which says where the bound comes
from). Pages and rows that no request owns hold NaN, padding rows of the output have to stay as they were."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from accelep_amd.capi import Batch, Buffer, RopeScaling, check, lib
from batch_helpers import NONE, Paged, dev, ints, packed_call, pool_of, want_batch
from long_context_helpers import assert_within, frequencies, rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


def say(*what):
    print(*what, flush=True)


def compare(x, got, window=0, rows=None):
    at, want, bound = x.want(window, rows)
    assert_within(got[at], want, bound)
    assert (got[sum(x.new):] == 3.0).all(), "padding rows were written"


KINDS = ["f32", "f16"]


# A step: one new token each, from none cached to several key ranges.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(9, 3, 64, 16), (8, 8, 128, 64), (8, 1, 128, 32), (20, 1, 64, 16),
                                                     (4, 2, 80, 16), (6, 2, 100, 128), (3, 3, 33, 16), (4, 1, 256, 256), (2, 2, 1, 16)])
def test_steps(kind, heads, kv_heads, dim, page):
    say("steps", kind, heads, kv_heads, dim, page)
    rng = np.random.default_rng(heads + dim)
    x = Paged(rng, [0, 1, 15, 16, 17, 31, 32, 63, 64, 255, 700, 3], [1] * 12, page, heads, kv_heads, dim, kind, pad=3)
    compare(x, x.call())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64])
def test_steps_over_long_ranges(kind, page):
    """Few requests, several thousand keys: their ranges are divided over workgroups."""
    rng = np.random.default_rng(11)
    x = Paged(rng, [9000, 5, 2047, 4500], [1] * 4, page, 8, 2, 128, kind)
    compare(x, x.call())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("longest", [None, 0, 1])
def test_chunks_beside_steps(kind, longest):
    """Requests without new tokens among them; longest known, not known and wrong."""
    rng = np.random.default_rng(12)
    x = Paged(rng, [300, 0, 17, 64, 1000, 5, 0, 130], [1, 140, 0, 65, 1, 2, 33, 1], 32, 8, 2, 64, kind, pad=5, longest=longest)
    compare(x, x.call())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (3, 3, 96), (4, 1, 256), (7, 1, 64), (4, 4, 30), (12, 4, 100)])
@pytest.mark.parametrize("window", [0, 1, 50, 200])
def test_chunks(kind, heads, kv_heads, dim, window):
    say("chunks", kind, heads, kv_heads, dim, window)
    rng = np.random.default_rng(heads + dim + window)
    x = Paged(rng, [0, 100, 333, 64], [70, 129, 50, 7], 16, heads, kv_heads, dim, kind, pad=1)
    rows = np.unique(np.concatenate([s + rng.integers(0, n, 12) for s, n in zip(x.starts, x.new)] + [x.starts[:-1], x.starts[1:] - 1]))
    compare(x, x.call(window), window, rows)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 16, 100, 1000, 1 << 40])
def test_steps_in_a_window(kind, window):
    rng = np.random.default_rng(window % 97)
    x = Paged(rng, [0, 14, 15, 16, 99, 100, 101, 2500], [1] * 8, 16, 6, 2, 64, kind)
    compare(x, x.call(window), window if window < 1 << 20 else 0)


@pytest.mark.parametrize("kind", KINDS)
def test_many_requests(kind):
    """More than a workgroup has threads, some without new tokens, one long among them."""
    rng = np.random.default_rng(13)
    seen = rng.integers(0, 40, 700)
    new = rng.integers(0, 3, 700)
    seen[333], new[333], new[500] = 5000, 1, 200
    x = Paged(rng, seen.tolist(), new.tolist(), 16, 2, 1, 64, kind, pad=2)
    compare(x, x.call(), rows=rng.integers(0, x.rows, 150).tolist() + [int(x.starts[333])])


@pytest.mark.parametrize("kind", KINDS)
def test_nothing_to_do(kind):
    rng = np.random.default_rng(14)
    x = Paged(rng, [5, 9], [0, 0], 16, 2, 1, 64, kind, pad=4)
    assert (x.call() == 3.0).all()
    x = Paged(rng, [], [], 16, 2, 1, 64, kind, pad=4)
    assert (x.call() == 3.0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_queries_in_rows_of_a_projection(kind):
    """Rows apart, from memory that is not aligned to 16 bytes."""
    rng = np.random.default_rng(15)
    for stride, shift in ((8 * 64 + 12, 0), (8 * 64 + 3, 1)):
        x = Paged(rng, [3, 50], [40, 1], 16, 8, 2, 64, kind)
        whole = np.full(x.rows * stride + shift, np.nan, np.float32)
        for i in range(x.rows):
            whole[shift + i * stride:shift + i * stride + 512] = x.q[i].ravel()
        d = dev(whole)
        out = dev(np.full((x.rows, 8, 64), 3.0, np.float32))
        check(lib().accel_hip_attention_paged(Buffer(d.at(shift), 4 * (len(whole) - shift), 0), C.byref(x.cache), C.byref(x.batch),
                                              out.buffer, 8, stride, 0))
        compare(x, out.numpy())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 33])
def test_pages_and_output_that_are_not_aligned(kind, dim):
    rng = np.random.default_rng(16)
    x = Paged(rng, [3, 70], [20, 1], 16, 4, 2, dim, kind)
    each = x.planes["k"].itemsize
    moved = {n: dev(np.concatenate([np.zeros(1, x.planes[n].dtype), x.planes[n].ravel()])) for n in "kv"}
    x.cache.k, x.cache.v = (Buffer(moved[n].ptr + each, x.planes[n].nbytes, 0) for n in "kv")
    out, qd = dev(np.full(x.rows * 4 * dim + 1, 3.0, np.float32)), dev(x.q)
    check(lib().accel_hip_attention_paged(qd.buffer, C.byref(x.cache), C.byref(x.batch), Buffer(out.at(1), 4 * x.rows * 4 * dim, 0),
                                          4, 0, 0))
    got = out.numpy()
    assert got[0] == 3.0
    compare(x, got[1:].reshape(x.rows, 4, dim))


# ---- what is not finite, and what has no page ----------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("plane", "kv")
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("seen,new", [(40, 5), (40, 70), (600, 1), (0, 200)])
def test_a_token_that_is_not_finite_reaches_the_rows_that_see_it(kind, plane, value, seen, new):
    """With a window: a token in the middle of the new ones (or of the old) is seen by some rows."""
    rng = np.random.default_rng(17)
    window = 64
    x = Paged(rng, [20, seen, 33], [3, new, 1], 16, 4, 2, 64, kind)
    token = seen + new // 2 if new > 1 else seen - 10
    d = x.planes[plane]
    at = int(x.table[1, token // 16]) * 16 + token % 16
    d[at, 1, 63] = value  # of key head 1 alone
    x.d[plane].upload(d)
    got = x.call(window)
    p = seen + np.arange(new)
    hit = (token <= p) & (token > p - window)
    rows = x.starts[1] + np.flatnonzero(hit)
    assert hit.any() and np.isnan(got[rows][:, 2:]).all()
    x.k[1], x.v[1] = x.k[1].copy(), x.v[1].copy()
    got[rows[:, None], [[2, 3]]] = 0
    at, want, bound = x.want(window)
    want[np.isin(at, rows)[:, None] & (np.arange(4) >= 2)[None, :]] = 0
    assert_within(got[at], want, bound)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("entry", [-1, 1 << 20, "width"])
@pytest.mark.parametrize("new", [1, 60])
def test_a_token_without_a_page(kind, entry, new):
    """The rows that see it are NaN, and no other; nothing outside the cache is read."""
    rng = np.random.default_rng(18)
    x = Paged(rng, [20, 40], [2, new], 16, 4, 2, 64, kind)
    if entry == "width":
        x.table = x.table[:, :3].copy()  # room for 48 tokens
        x.width, first = 3, 48
    else:
        x.table[1, 2], first = entry, 32
    x.upload()
    got = x.call()
    p = 40 + np.arange(new)
    bad = x.starts[1] + np.flatnonzero(p >= first)
    assert np.isnan(got[bad]).all()
    at, want, bound = x.want(rows=np.setdiff1d(np.arange(x.rows), bad))
    assert_within(got[at], want, bound)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_query_that_is_not_finite_stays_alone(kind, value):
    rng = np.random.default_rng(19)
    x = Paged(rng, [20, 40], [40, 1], 16, 4, 2, 64, kind)
    x.q[7, 1, 5] = x.q[40, 3, 0] = value
    got = x.call()
    assert np.isnan(got[7, 1]).all() and np.isnan(got[40, 3]).all()
    x.q[7, 1, 5] = x.q[40, 3, 0] = 0
    at, want, bound = x.want()
    for r, h in ((7, 1), (40, 3)):
        got[r, h] = want[r, h] = 0
    assert_within(got[at], want, bound)


@pytest.mark.parametrize("kind", KINDS)
def test_lengths_and_starts_out_of_range(kind):
    """What device memory holds may be wrong: rows stay inside the batch, tokens inside the table."""
    rng = np.random.default_rng(20)
    x = Paged(rng, [20, 40, 5], [30, 1, 4], 16, 4, 2, 64, kind, pad=2)
    good = x.call()
    x.d["seen"].upload(np.array([20, 2 ** 31 - 1, -5], np.int32))
    got = x.call()
    np.testing.assert_array_equal(got[:30], good[:30])
    assert np.isnan(got[30]).all() and (got[35:] == 3.0).all()
    x.d["seen"].upload(np.array([20, 40, 5], np.int32))
    for starts in ([-7, 30, 31, 35], [0, 30, 31, 2 ** 31 - 1], [30, 30, 31, 20], [5, 2, 2 ** 31 - 1, -1]):
        x.d["starts"].upload(np.array(starts, np.int32))
        x.call()
    x.d["starts"].upload(x.starts)
    np.testing.assert_array_equal(x.call(), good)


# ---- ranges of values ----------------------------------------------------------------------------

@pytest.mark.parametrize("kind,low,high", [("f32", -100, 20), ("f32", -3, 3), ("f32", -40, 40), ("f16", -14, 12), ("f16", -24, -10)])
@pytest.mark.parametrize("new", [1, 40])
def test_rows_of_many_magnitudes(kind, low, high, new):
    """Values of 2^low .. 2^high, other powers in every token; queries that bring the scores to a few units."""
    rng = np.random.default_rng(high - low)

    def make(name, r, total):
        x = rng.standard_normal((total, 2, 64))
        return x * np.exp2(rng.integers(low, high + 1, (total, 1, 1))) if name == "v" else x

    x = Paged(rng, [70, 300], [new, 1], 16, 8, 2, 64, kind, make=make)
    at, want, bound = x.want()
    # A weight has 22 bits down to 2^-6 of the largest weight * value, and an f16 value is exact: what the sums lose is
    # 2^-24 of the largest value a row sees, once for each key.
    big = np.array([max(np.abs(v.astype(np.float64)).max() for v in x.v)])
    assert_within(x.call()[at], want, bound + 2.0 ** -24 * 300 * big * 2.0 ** -3)


@pytest.mark.parametrize("new", [1, 40])
def test_values_near_the_largest_float(new):
    """Their weighted mean is one, their sum is not."""
    rng = np.random.default_rng(21)
    x = Paged(rng, [500, 30], [new, 1], 16, 4, 2, 64, "f32",
              make=lambda name, r, total: rng.standard_normal((total, 2, 64)) if name == "k" else np.full((total, 2, 64), 3.3e38))
    got = x.call()
    np.testing.assert_allclose(got, 3.3e38, rtol=1e-5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_queries_of_any_size(kind, new, scale):
    """Tiny queries weigh all keys the same; huge ones pick the key with the largest score (or, past the largest float, NaN)."""
    rng = np.random.default_rng(22)
    x = Paged(rng, [100], [new], 16, 4, 2, 64, kind)
    x.q = (x.q * scale).astype(np.float32)
    at, want, bound = x.want()
    got = x.call()
    if scale < 1:
        assert_within(got[at], want, bound)
    else:
        np.testing.assert_allclose(got[at], want, rtol=1e-5, atol=1e-6)


# ---- packed prompts ------------------------------------------------------------------------------

@pytest.mark.parametrize("lengths,heads,kv_heads,dim,window", [
    ([1], 2, 1, 64, 0), ([1, 1, 1], 9, 3, 64, 0), ([5, 0, 17, 16, 33], 9, 3, 64, 0), ([128, 129, 127], 4, 4, 128, 0),
    ([300, 7], 8, 2, 128, 0), ([200, 100], 8, 2, 128, 30), ([65, 64, 1], 6, 2, 80, 0), ([40, 90], 4, 1, 256, 0),
    ([130, 20], 4, 2, 100, 64), ([50, 31], 3, 3, 33, 0), ([90, 5], 16, 1, 96, 1), ([2, 3], 20, 1, 64, 0)])
def test_packed(lengths, heads, kv_heads, dim, window):
    say("packed", lengths, heads, kv_heads, dim, window)
    rng = np.random.default_rng(sum(lengths) + dim)
    starts = np.concatenate([[0], np.cumsum(lengths)])
    n, pad = int(starts[-1]), 3
    q = (2 * rng.standard_normal((n + pad, heads, dim))).astype(np.float32)
    k, v = (rng.standard_normal((n + pad, kv_heads, dim)).astype(np.float32) for _ in "kv")
    for x in (q, k, v):
        x[n:] = np.nan
    parts = [[x[a:b] for a, b in zip(starts, starts[1:])] for x in (k, v)]
    rows = None if n < 200 else np.unique(np.concatenate([starts[:-1], starts[1:] - 1, rng.integers(0, n, 60)]))
    at, want, bound = want_batch(q, *parts, [0] * len(lengths), starts, window, rows)
    for longest in {0, max(lengths), 1}:
        got = packed_call(q, k, v, starts, heads, kv_heads, dim, n + pad, window, longest=longest)
        assert_within(got[at], want, bound)
        assert (got[n:] == 3.0).all()


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dim", [64, 100])
def test_packed_in_rows_of_a_projection(shift, dim):
    """Queries, keys and values as parts of the same rows, aligned to 16 bytes or not."""
    rng = np.random.default_rng(23)
    lengths, heads, kv = [60, 1, 140], 8, 2
    starts = np.concatenate([[0], np.cumsum(lengths)])
    n, width = int(starts[-1]), (heads + 2 * kv) * dim + shift
    whole = rng.standard_normal((n, width)).astype(np.float32)
    flat = np.concatenate([np.zeros(shift, np.float32), whole.ravel()])
    d = dev(flat)
    q, k, v = (whole[:, a * dim:b * dim].reshape(n, -1, dim) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    parts = [Buffer(d.at(shift + at * dim), 4 * (len(flat) - shift - at * dim), 0) for at in (0, heads, heads + kv)]
    got = packed_call(*parts, starts, heads, kv, dim, n, row_stride=width, kv_stride=width)
    at, want, bound = want_batch(q, [k[a:b] for a, b in zip(starts, starts[1:])], [v[a:b] for a, b in zip(starts, starts[1:])],
                                 [0, 0, 0], starts, 0, np.arange(0, n, 7))
    assert_within(got[at], want, bound)


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("plane", "kv")
def test_a_prompt_does_not_reach_another(value, plane):
    """Nor does what lies behind the last row reach the last prompt."""
    rng = np.random.default_rng(24)
    lengths = [50, 40, 150, 3]
    starts = np.concatenate([[0], np.cumsum(lengths)])
    n = int(starts[-1])
    q, k, v = (rng.standard_normal((n + 40, h, 64)).astype(np.float32) for h in (4, 2, 2))
    clean = packed_call(q, k, v, starts, 4, 2, 64, n + 40)
    x = {"k": k.copy(), "v": v.copy()}
    x[plane][[50, 89, 95, n, n + 20]] = value
    got = packed_call(q, x["k"], x["v"], starts, 4, 2, 64, n + 40)
    assert np.isnan(got[50:90]).all() and np.isnan(got[95:240]).all()
    for a, b in ((0, 50), (240, n)):
        np.testing.assert_array_equal(got[a:b], clean[a:b])
    at, want, bound = want_batch(q, [k[90:240]], [v[90:240]], [0], [90, 240], 0, np.arange(90, 95))
    assert_within(got[at], want, bound)


# ---- a run of all of them ------------------------------------------------------------------------

def test_requests_served_together():
    """Four requests through three steps of one layer, replayed from a graph: tables, scaled rotary positions at the
    rows' positions, keys and values into their slots, attention. A prompt, then single tokens; one request ends and
    a new one takes its place and its pages."""
    rng = np.random.default_rng(25)
    heads, kv, dim, page, requests, rows, width = 6, 2, 64, 16, 4, 96, 8
    L, row = lib(), (heads + 2 * kv) * dim
    f = frequencies(1, dim)
    fd = dev(f)
    d = {n: ints(x) for n, x in {"counts": [0] * 4, "lengths": [0] * 4, "seen": [0] * 4, "starts": [0] * 5,
                                 "table": np.full((4, width), -1), "slots": [0] * rows, "positions": [0] * rows}.items()}
    pool, held = pool_of(rng.permutation(14), 14, page)
    batch = Batch(d["seen"].buffer, d["starts"].buffer, d["table"].buffer, requests, rows, width, 0)
    from accelep_amd.capi import CACHE_F32, CachePaged
    planes = [dev(np.full((14, page, kv, dim), np.nan, np.float32)) for _ in "kv"]
    cache = CachePaged(planes[0].buffer, planes[1].buffer, CACHE_F32, 14, page, kv, dim)
    x, out = dev(np.zeros((rows, row), np.float32)), dev(np.zeros((rows, heads, dim), np.float32))
    part = lambda at: Buffer(x.at(at * dim), 4 * (rows * row - at * dim), 0)  # noqa: E731

    def step():
        check(L.accel_hip_batch_tables(d["counts"].buffer, d["lengths"].buffer, C.byref(pool), C.byref(batch), d["slots"].buffer,
                                       d["positions"].buffer, d["lengths"].buffer, held[1].buffer))
        check(L.accel_hip_rope_scaled(x.buffer, x.buffer, fd.buffer, d["positions"].buffer, rows, heads + kv, dim, row, dim, 0, 0, 1.0))
        check(L.accel_hip_append_paged(part(heads), part(heads + kv), C.byref(cache), d["slots"].buffer, rows, row))
        check(L.accel_hip_attention_paged(x.buffer, C.byref(cache), C.byref(batch), out.buffer, heads, row, 0))

    step()  # no tokens: grows what has to grow
    graph = C.c_void_p()
    check(L.accel_hip_capture_begin())
    step()
    check(L.accel_hip_capture_end(C.byref(graph)))
    past = [[[], []] for _ in range(requests)]
    try:
        for counts, keep in (([40, 1, 0, 33], None), ([1, 1, 20, 1], None), ([1, 50, 1, 2], [0, 2, 20, 30]), ([1, 1, 1, 1], None)):
            if keep is not None:
                kd = ints(keep)
                check(L.accel_hip_release_pages(kd.buffer, d["lengths"].buffer, C.byref(pool), C.byref(batch)))
                for r in range(requests):
                    past[r] = [p[:keep[r]] for p in past[r]]
            fresh = rng.standard_normal((rows, row)).astype(np.float32)
            x.upload(fresh)
            d["counts"].upload(np.array(counts, np.int32))
            out.upload(np.full((rows, heads, dim), 3.0, np.float32))
            check(L.accel_hip_graph_launch(graph, 1))
            got = out.numpy()
            assert held[1].numpy()[1] == 0
            turned = x.numpy()  # what the rotation gave: compared on its own, and taken as it is for the rest
            at = 0
            for r, n in enumerate(counts):
                mine = slice(at, at + n)
                seen = len(past[r][0])
                p = seen + np.arange(n)
                want, bound = rotated(fresh[mine, :(heads + kv) * dim].reshape(n, heads + kv, dim), f, p, 0, 1.0)
                assert_within(turned[mine, :(heads + kv) * dim].reshape(n, heads + kv, dim), want, bound)
                new = turned[mine].reshape(n, heads + 2 * kv, dim)
                past[r][0] = [*past[r][0], *new[:, heads:heads + kv]]
                past[r][1] = [*past[r][1], *new[:, heads + kv:]]
                if n:
                    rows_at, want, bound = want_batch(new[:, :heads], [np.array(past[r][0])], [np.array(past[r][1])], [seen], [0, n], 0)
                    assert_within(got[mine], want, bound)
                at += n
            assert (got[at:] == 3.0).all()
            assert d["lengths"].numpy().tolist() == [len(p[0]) for p in past]
    finally:
        check(L.accel_hip_graph_destroy(graph))
    owned = d["table"].numpy()
    free = held[0].numpy()[:held[1].numpy()[0]]
    assert sorted([*owned[owned >= 0], *free]) == list(range(14))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 40])
def test_captured_and_replayed_while_requests_grow(kind, new):
    """The lengths are in device memory: a graph of one step serves the later ones. Eager calls come between."""
    rng = np.random.default_rng(26)
    x = Paged(rng, [3000, 20, 600], [new] * 3, 16, 8, 2, 64, kind)
    final = list(x.seen)
    qd, out = dev(x.q), dev(np.zeros((x.rows, 8, 64), np.float32))
    call = lambda: x.call(q=qd, out=out)  # noqa: E731
    call()
    graph = C.c_void_p()
    L = lib()
    check(L.accel_hip_capture_begin())
    check(L.accel_hip_attention_paged(qd.buffer, C.byref(x.cache), C.byref(x.batch), out.buffer, 8, 0, 0))
    check(L.accel_hip_capture_end(C.byref(graph)))
    try:
        for shorter in (2900, 1000, 0, 30):
            x.seen = [max(0, s - shorter) for s in final]
            x.d["seen"].upload(np.asarray(x.seen, np.int32))
            eager = call()
            out.upload(np.zeros((x.rows, 8, 64), np.float32))
            check(L.accel_hip_graph_launch(graph, 2))
            replayed = out.numpy()
            np.testing.assert_array_equal(replayed, eager)
            k, v = ([p[:s + new] for p, s in zip(y, x.seen)] for y in (x.k, x.v))
            at, want, bound = want_batch(x.q, k, v, x.seen, x.starts, 0, x.starts[:-1])
            assert_within(replayed[at], want, bound)
    finally:
        check(L.accel_hip_graph_destroy(graph))


@pytest.mark.parametrize("kind", KINDS)
def test_the_same_call_gives_the_same_bits(kind):
    rng = np.random.default_rng(27)
    x = Paged(rng, [3000, 20, 600], [1, 40, 1], 16, 8, 2, 64, kind)
    first = x.call()
    for _ in range(3):
        np.testing.assert_array_equal(x.call(), first)
