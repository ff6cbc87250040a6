"""Windowed attention where values of far magnitudes meet: large ones of little weight."""

from __future__ import annotations

import numpy as np
import pytest

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
