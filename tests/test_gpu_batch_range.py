"""Attention of a batch where values of far magnitudes meet, against 64-bit softmax attention, each row bounded by what it
sees itself."""

from __future__ import annotations

import numpy as np
import pytest

from batch_helpers import Paged, check, lib
from long_context_helpers import assert_within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    check(lib().accel_hip_init())
    yield


def keys_below(rng, total, at, power):
    """Keys of scores around 0 with the queries of `queries`, but for the tokens `at`, whose lie at log2 units of `power`."""
    k = rng.standard_normal((total, 2, 64))
    k[:, :, 0] = 0
    k[at, :, 0] = np.asarray(power, np.float64)[:, None] * np.log(2)
    return k


def queries(x):
    x.q /= 16
    x.q[:, :, 0] = 8  # sqrt(64): the first dim of a key is its score


# ---- few rows over fp32 --------------------------------------------------------------------------

@pytest.mark.parametrize("power", [-30, -39, -41, -60, -75, -80, -90, -110])
@pytest.mark.parametrize("seen,new", [(60, 1), (500, 4), (9000, 1)])
def test_a_large_value_of_little_weight(power, seen, new):
    """2^126 with a weight of 2^power of the others' decides the row, and keeps its bits."""
    rng = np.random.default_rng(-power + seen)
    for at in (1, seen // 2, seen - 1):
        def make(name, r, total, at=at):
            if name == "k":
                return keys_below(rng, total, [at], [power])
            v = rng.standard_normal((total, 2, 64))
            v[at] = 2.0 ** 126 * rng.uniform(-1, 1, (2, 64))
            return v

        x = Paged(rng, [seen], [new], 16, 4, 2, 64, "f32", make=make)
        queries(x)
        rows, want, bound = x.want()
        assert_within(x.call()[rows], want, bound, floor=0)


@pytest.mark.parametrize("seen,new", [(60, 1), (500, 4), (9000, 1)])
def test_large_values_of_all_weights(seen, new):
    """One of 2^97 that weighs as much as the others, some of 2^126 that weigh from 2^-25 to 2^-95 of that, in one row."""
    rng = np.random.default_rng(seen)
    at = np.sort(rng.permutation(seen)[:9])
    powers = [0, -25, -35, -45, -55, -65, -75, -85, -95]
    for order in (1, -1):
        for left_out in range(8):  # so that each of them is the largest share of a row once
            keep = at[left_out:]
            levels = powers[left_out:][::order]

            def make(name, r, total, keep=keep, levels=levels):
                if name == "k":
                    return keys_below(rng, total, keep, levels)
                v = rng.standard_normal((total, 2, 64))
                v[keep] = np.where(np.array(levels) == 0, 2.0 ** 97, 2.0 ** 126)[:, None, None] * rng.uniform(-1, 1, (len(keep), 2, 64))
                return v

            x = Paged(rng, [seen], [new], 16, 4, 2, 64, "f32", make=make)
            queries(x)
            rows, want, bound = x.want()
            assert_within(x.call()[rows], want, bound, floor=0)
