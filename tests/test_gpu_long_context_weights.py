"""Windowed attention where values of far magnitudes meet: large ones of little weight, rows of zeros beside small ones."""

from __future__ import annotations

import numpy as np
import pytest

from long_context_dispatch import F32, many
from long_context_helpers import assert_within, attend, attention_window_call, check, lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


def queries_and_keys(r, seq, length, heads, at, powers):
    """Scores around 0, but for the keys `at`, whose lie at log2 units of `powers`: the first dim of a key is its score."""
    q, k, v = (r.standard_normal((n, heads, 64)) for n in (seq, length, length))
    q /= 16
    q[:, :, 0] = 8
    k[:, :, 0] = 0
    k[at, :, 0] = np.asarray(powers, np.float64)[:, None] * np.log(2)
    return q.astype(np.float32), k.astype(np.float32), v


@pytest.mark.parametrize("power", [-30, -39, -41, -60, -75, -80, -90, -110])
@pytest.mark.parametrize("seq,length", [(1, 60), (4, 500), (1, 9000)])
def test_a_large_value_of_little_weight(power, seq, length):
    """2^126 with a weight of 2^power of the others' decides the row, and keeps its bits."""
    r = np.random.default_rng(-power + length)
    for at in (1, length // 2, length - seq - 1):
        q, k, v = queries_and_keys(r, seq, length, 2, [at], [power])
        v[at] = 2.0 ** 126 * r.uniform(-1, 1, (2, 64))
        v = v.astype(np.float32)
        want, bound = attend(q, k, v, length - seq, 0, 0)
        assert_within(attention_window_call(q, k, v, length - seq), want, bound, floor=0)


@pytest.mark.parametrize("seq,length", [(1, 60), (4, 500), (1, 9000)])
def test_large_values_of_all_weights(seq, length):
    """One of 2^97 that weighs as much as the others, some of 2^126 that weigh from 2^-25 to 2^-95 of that, in one row."""
    r = np.random.default_rng(length)
    at = np.sort(r.permutation(length - seq)[:9])
    powers = np.array([0, -25, -35, -45, -55, -65, -75, -85, -95])
    for order in (1, -1):
        for left_out in range(8):  # so that each of them is the largest share of a row once
            keep, levels = at[left_out:], powers[left_out:][::order]
            q, k, v = queries_and_keys(r, seq, length, 2, keep, levels)
            v[keep] = np.where(levels == 0, 2.0 ** 97, 2.0 ** 126)[:, None, None] * r.uniform(-1, 1, (len(keep), 2, 64))
            v = v.astype(np.float32)
            want, bound = attend(q, k, v, length - seq, 0, 0)
            assert_within(attention_window_call(q, k, v, length - seq), want, bound, floor=0)


@pytest.mark.parametrize("power", [-116, -60, -30, -12, -8, 0, 30])
@pytest.mark.parametrize("zeros", [[0], [5, 6, 40], list(range(32)), list(range(64, 99))])
@pytest.mark.parametrize("score", [0, 12])
def test_rows_of_zeros_beside_small_values(power, zeros, score):
    """Many rows. A value row of zeros adds nothing to a row's sum, so the others keep their bits, also where it has the
    largest weight."""
    r = np.random.default_rng(len(zeros) + score)
    seq, length, copies = 70, 300, 512
    q, k, v = queries_and_keys(r, seq, length, 2, zeros, [score] * len(zeros))
    v *= 2.0 ** power
    v[zeros] = 0
    v = v.astype(np.float32)
    some = np.arange(0, seq, 9)
    want, bound = attend(q, k, v, length - seq, 0, 0, some)
    got = attention_window_call(many(q, copies, F32, length - seq, 2), k, v, length - seq)
    # Beside what `attend` counts, a second part of a weight or value that is no normal f16 number: 2^-25 where the largest
    # weight * value row holds 2^3 * 2^3 at least in these units, so 2^-28 of the largest a key for the weight, and the same
    # for the value; four times that is allowed. An output below 2^-126 is rounded to 2^-149.
    p = np.exp(np.einsum("shd,thd->sht", q[some].astype(np.float64), k.astype(np.float64)) / 8)
    p[np.arange(length)[None, None, :] > (length - seq + some)[:, None, None] + np.zeros((1, 2, 1))] = 0
    p /= p.sum(axis=2, keepdims=True)
    largest = (p * np.abs(v).max(axis=2).T[None]).max(axis=2)
    bound += 2.0 ** -25 * length * largest[..., None]
    if power < -100:
        # A weight meets its value row's scale, 2^-127 at least, in one fp32 product: where that is below 2^-126 it is off by
        # 2^-150, 2^-23 of the largest weight, which is 1 at least in these units. (22 bits of the largest are promised.)
        bound += 2.0 ** -23 * p.max(axis=2)[..., None] * np.abs(v.astype(np.float64)).sum(axis=0)
    assert_within(got[some, ::copies], want, bound, floor=2.0 ** -149)
