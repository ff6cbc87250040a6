"""Attention over keys and values near the ends of fp32's range: what is finite in 64 bits and fits fp32 comes out so."""

from __future__ import annotations

import numpy as np
import pytest

from long_context_dispatch import F32, Q8, many, takes_many_rows
from long_context_helpers import (Cache, assert_within, attend, attention_q8_call, attention_window_call, check, lib,
                                  sees)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


# (seq, length, copies): few rows over a range in one part and in several; many rows, the same.
SIZES = [(3, 50, 1), (2, 9000, 1), (17, 30000, 16), (200, 600, 512)]
SIZE_IDS = ["few", "few-long", "many-divided", "many"]


@pytest.mark.parametrize("seq,length,copies", SIZES, ids=SIZE_IDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 4)])
@pytest.mark.parametrize("large", [100, 119])
def test_window_attention_of_large_keys_and_small_queries(seq, length, copies, window, sinks, large):
    """Keys of 2^large and more with queries that make ordinary scores of them: rows of scales of their own."""
    r = np.random.default_rng(41)
    position = length - seq
    while copies > 1 and not takes_many_rows(F32, seq, position, 2 * copies, 2, window, sinks):
        copies *= 2  # a window is short
    q, k, v = (r.standard_normal(s).astype(np.float32) for s in ((seq, 2, 64), (length, 2, 64), (length, 2, 64)))
    q *= np.float32(2.0 ** -large)
    k *= (2.0 ** (large + r.integers(-2, 5, (length, 2, 1)))).astype(np.float32)
    some = np.unique(np.r_[0:seq:7, seq - 1])
    want, bound = attend(q, k, v, position, window, sinks, some)
    got = attention_window_call(many(q, copies, F32, position, 2, window, sinks), k, v, position, window, sinks)
    assert_within(got[some, ::copies], want, bound)


@pytest.mark.parametrize("seq,length,copies", SIZES, ids=SIZE_IDS)
@pytest.mark.parametrize("block", [1, 16, 64])
@pytest.mark.parametrize("large", [100, 119])
def test_attention_q8_of_large_keys_and_small_queries(seq, length, copies, block, large):
    r = np.random.default_rng(42)
    position = length - seq
    cache = Cache(length, 2, 64, block)
    cache.fill(r, length)
    cache.scale["k"] *= np.float32(2.0 ** large)
    cache.upload()
    q = (r.standard_normal((seq, 2, 64)) * 2.0 ** -large).astype(np.float32)
    some = np.unique(np.r_[0:seq:7, seq - 1])
    want, bound = attend(q, cache.values("k"), cache.values("v"), position, 0, 0, some, cache.value_scale(length))
    got = attention_q8_call(many(q, copies, Q8, position, 2), cache, position)
    assert_within(got[some, ::copies], want, bound)


def large_values(r, shape, signs):
    """Between a third and nearly all of the largest float."""
    x = r.uniform(1.2e38, 3.3e38, shape)
    return (x * r.choice([-1.0, 1.0], shape) if signs else x).astype(np.float32)


@pytest.mark.parametrize("seq,length,copies", SIZES, ids=SIZE_IDS)
@pytest.mark.parametrize("dim", [64, 100, 128, 256])
@pytest.mark.parametrize("signs", [False, True])
def test_window_attention_of_values_near_the_largest_float(seq, length, copies, dim, signs):
    """The sum over the keys of weight times value passes the largest float, its quotient does not."""
    r = np.random.default_rng(43)
    position = length - seq
    q, k = (r.standard_normal(s).astype(np.float32) for s in ((seq, 2, dim), (length, 2, dim)))
    v = large_values(r, (length, 2, dim), signs)
    some = np.unique(np.r_[0:seq:13, seq - 1])
    want, bound = attend(q, k, v, position, 0, 0, some)
    got = attention_window_call(many(q, copies, F32, position, 2), k, v, position)
    assert_within(got[some, ::copies], want, bound)


@pytest.mark.parametrize("seq,length,copies", SIZES, ids=SIZE_IDS)
@pytest.mark.parametrize("block", [1, 4, 16, 64])
@pytest.mark.parametrize("dim", [64, 100, 128, 256])
def test_attention_q8_of_values_near_the_largest_float(seq, length, copies, block, dim):
    r = np.random.default_rng(44)
    position = length - seq
    cache = Cache(length, 2, dim, block)
    cache.fill(r, length)
    cache.codes["v"][:] = r.integers(80, 128, cache.codes["v"].shape)
    cache.codes["v"][:, :, ::5] *= -1
    cache.scale["v"][:] = r.uniform(1.3e36, 2.6e36, cache.scale["v"].shape)
    cache.upload()
    q = r.standard_normal((seq, 2, dim)).astype(np.float32)
    some = np.unique(np.r_[0:seq:13, seq - 1])
    want, bound = attend(q, cache.values("k"), cache.values("v"), position, 0, 0, some, cache.value_scale(length))
    got = attention_q8_call(many(q, copies, Q8, position, 2), cache, position)
    assert_within(got[some, ::copies], want, bound)


@pytest.mark.parametrize("seq,length,copies", SIZES[1:], ids=SIZE_IDS[1:])
@pytest.mark.parametrize("block", [1, 4, 16, 64])
@pytest.mark.parametrize("rise", [2.0, 5.0])
@pytest.mark.parametrize("first", [1.0, 2.0 ** -90])
def test_attention_q8_of_large_values_behind_keys_of_lower_scores(seq, length, copies, block, rise, first):
    """Scores rise by less than 8 in log2 units halfway, so the weights behind pass 1; the values there are near the
    largest float, and before ordinary ones (or 2^-90 times those). Over many parts only one of them has the rise."""
    r = np.random.default_rng(45)
    position = length - seq
    cache = Cache(length, 1, 64, block)
    cache.fill(r, length)
    middle = length // 2 // 64 * 64 - 64
    cache.codes["k"][:, 0, 0] = 1
    cache.codes["k"][middle:, 0, 0] = 127
    cache.scale["k"][:] = 1 / 127
    cache.scale["v"][:] = first * r.uniform(0.5, 1, cache.scale["v"].shape) / 64
    cache.scale["v"][middle // block:] = r.uniform(1.3e36, 2.6e36, cache.scale["v"][middle // block:].shape)
    cache.upload()
    q = (r.standard_normal((seq, 2, 64)) / 64).astype(np.float32)
    q[:, :, 0] = 8 * rise * 127 / 126
    some = np.unique(np.r_[0:seq:13, seq - 1])
    want, bound = attend(q, cache.values("k"), cache.values("v"), position, 0, 0, some, cache.value_scale(length))
    got = attention_q8_call(many(q, copies, Q8, position, 1), cache, position)
    assert_within(got[some, ::copies], want, bound)


@pytest.mark.parametrize("seq,heads,length", [(1, 2, 70), (7, 4, 300), (16, 2, 5000)])
@pytest.mark.parametrize("small", [1.0, 2.0 ** -100])
def test_rows_of_one_tile_that_see_large_values_and_that_do_not(seq, heads, length, small):
    """A window of 5: the key before the last rows' own holds values near the largest float; rows that do not see it
    keep the bits of theirs, those that do have a finite quotient."""
    r = np.random.default_rng(46)
    position = length - seq
    q, k, v = (r.standard_normal(s).astype(np.float32) for s in ((seq, heads, 64), (length, 2, 64), (length, 2, 64)))
    v *= np.float32(small)
    for t in sorted({length - 2, position + seq // 2, max(0, position - 3)}):
        vv = v.copy()
        vv[t] = large_values(r, (2, 64), True)
        want, bound = attend(q, k, vv, position, 5, 1)
        got = attention_window_call(q, k, vv, position, 5, 1)
        assert_within(got, want, bound, floor=0)


def test_small_values_beside_a_large_one_that_counts_for_nothing():
    """A visible key whose values are near the largest float and whose weight is e^-100 of the others'."""
    r = np.random.default_rng(47)
    for seq, length in ((1, 60), (3, 4000)):
        q, k, v = (r.standard_normal(s).astype(np.float32) for s in ((seq, 2, 64), (length, 1, 64), (length, 1, 64)))
        q /= 8
        q[:, :, 0] = 400
        k[:, 0, 0] = 1
        for t in (0, length // 2, length - seq):
            kk, vv = k.copy(), v.copy()
            kk[t, 0, 0] = -1
            vv[t] = large_values(r, (1, 64), True)
            want, bound = attend(q, kk, vv, length - seq, 0, 0)
            assert_within(attention_window_call(q, kk, vv, length - seq), want, bound)


@pytest.mark.parametrize("seq,heads,kv_heads,copies", [(1, 128, 128, 1), (2, 4, 1, 1), (40, 2, 1, 256)])
@pytest.mark.parametrize("rise", [200.0, 4000.0])
@pytest.mark.parametrize("small", [1.0, 2.0 ** -100])
def test_small_values_behind_large_ones_whose_weights_vanish(seq, heads, kv_heads, copies, rise, small):
    """The first keys' values are near the largest float; scores rise by `rise` over 4000 keys, so what they gave
    the sum fades, slowly or at once, and only the last keys count."""
    r = np.random.default_rng(48)
    length = 4000
    q, k, v = (r.standard_normal(s).astype(np.float32) for s in ((seq, heads, 64), (length, kv_heads, 64), (length, kv_heads, 64)))
    v *= np.float32(small)
    v[:200] = large_values(r, (200, kv_heads, 64), True)
    q[:, :, 0] = 8
    k[:, :, 0] = np.linspace(0, rise, length)[:, None]
    want, bound = attend(q, k, v, length - seq, 0, 0)
    got = attention_window_call(many(q, copies, F32, length - seq, kv_heads), k, v, length - seq)
    assert_within(got[:, ::copies], want, bound, floor=0)


def winners(q, k, position, window=0, sinks=0):
    """Of each row and head the visible key of the largest score, and whether no rounding of scores can change it: the
    next score is further below than all they may be off by (2^-14 of the largest sum of |q k|), and 2^10 besides."""
    seq, heads, dim = q.shape
    group = heads // k.shape[1]
    seen = sees(position, seq, len(k), window, sinks)
    best, sure = np.zeros((seq, heads), int), np.zeros((seq, heads), bool)
    for h in range(heads):
        kk, qq = k[:, h // group].astype(np.float64), q[:, h].astype(np.float64)
        x = np.where(seen, qq @ kk.T / np.sqrt(dim), -np.inf)
        off = (np.where(seen, np.abs(qq) @ np.abs(kk).T, 0) / np.sqrt(dim)).max(axis=1) * 2.0 ** -14
        best[:, h] = x.argmax(axis=1)
        top = np.sort(x, axis=1)[:, -2:]
        sure[:, h] = top[:, 1] - top[:, 0] > off + 1024
    return best, sure


@pytest.mark.parametrize("seq,length,copies", [(40, 40, 1), (300, 300, 1), *SIZES, (600, 600, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 4)])
@pytest.mark.parametrize("large", [20, 30, 60, 115])
@pytest.mark.parametrize("block", [None, 1, 16, 64])
def test_scores_so_far_apart_that_one_key_wins(seq, length, copies, window, sinks, large, block):
    """Visible keys of 2^large with ordinary queries: each row's output is the values of its winner, whose score may be
    far below zero too (the first rows see one key)."""
    r = np.random.default_rng(49)
    position = length - seq
    pairs = F32 if block is None else Q8
    while copies > 1 and not takes_many_rows(pairs, seq, position, 2 * copies, 2, window, sinks):
        copies *= 2
    q = r.standard_normal((seq, 2, 64)).astype(np.float32)
    if block is None:
        k, v = (r.standard_normal((length, 2, 64)).astype(np.float32) for _ in "kv")
        k *= np.float32(2.0 ** large)
        got = attention_window_call(many(q, copies, pairs, position, 2, window, sinks), k, v, position, window, sinks)
    else:
        cache = Cache(length, 2, 64, block)
        cache.fill(r, length)
        cache.scale["k"] *= np.float32(2.0 ** large)
        cache.upload()
        k, v = cache.values("k"), cache.values("v")
        got = attention_q8_call(many(q, copies, pairs, position, 2, window, sinks), cache, position, window, sinks)
    best, sure = winners(q, k, position, window, sinks)
    assert sure.mean() > 0.9
    for h in range(2):
        want = v[best[:, h], h].astype(np.float64)
        # a weight and its values are cut by 1.5 * 2^-22 each (values of the row's largest) and the quotient rounds
        bound = 4 * 2.0 ** -22 * np.abs(want).max(axis=1, keepdims=True)
        assert_within(got[sure[:, h], h * copies], want[sure[:, h]], np.broadcast_to(bound, want.shape)[sure[:, h]], floor=0)
