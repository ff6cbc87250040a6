"""Attention of a batch where values of far magnitudes meet, against 64-bit softmax attention, each row bounded by what it
sees itself."""

from __future__ import annotations

import numpy as np
import pytest

from batch_helpers import Paged, check, lib, packed_call
from long_context_helpers import assert_within, attend

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


# ---- many rows over fp32 -------------------------------------------------------------------------

def seen_largest(x):
    """[row, head]: keys seen, times the largest weight * (largest magnitude of its value row)."""
    out = np.zeros((len(x.q), x.heads))
    group = x.heads // x.kv_heads
    for r, seen in enumerate(x.seen):
        k, v = x.k[r].astype(np.float64), np.abs(x.v[r].astype(np.float64)).max(axis=2)
        for i in range(x.new[r]):
            n = seen + i + 1
            for h in range(x.heads):
                s = k[:n, h // group] @ x.q[x.starts[r] + i, h].astype(np.float64) / np.sqrt(x.dim)
                p = np.exp(s - s.max())
                out[x.starts[r] + i, h] = n * (p / p.sum() * v[:n, h // group]).max()
    return out


def compare_many(x, window=0):
    # Beside what `attend` counts, a second part of a weight or value that is no normal f16 number: 2^-25 where the largest
    # weight * value row holds 2^3 * 2^3 at least in these units, so 2^-28 of the largest a key for the weight, and the same
    # for the value; four times that is allowed. An output below 2^-126 is rounded to 2^-149.
    rows, want, bound = x.want(window)
    assert_within(x.call(window)[rows], want, bound + 2.0 ** -25 * seen_largest(x)[rows][..., None], floor=2.0 ** -149)


@pytest.mark.parametrize("power", [-90, -104, -108, -112, -116, -124])
@pytest.mark.parametrize("seen,new", [([0, 30], [70, 40]), ([3000], [50])])
def test_tiny_values(power, seen, new):
    """All about 2^power: 22 bits of each."""
    rng = np.random.default_rng(-power)
    x = Paged(rng, seen, new, 16, 4, 2, 64, "f32",
              make=lambda name, r, total: rng.standard_normal((total, 2, 64)) * (1 if name == "k" else 2.0 ** power))
    compare_many(x)


@pytest.mark.parametrize("power", [-116, -108, -90])
def test_tiny_values_of_packed_prompts(power):
    rng = np.random.default_rng(-power)
    q, k, v = (rng.standard_normal((110, h, 64)).astype(np.float32) for h in (4, 2, 2))
    v *= np.float32(2.0 ** power)
    want, bound = attend(q, k, v, 0, 0, 0)
    assert_within(packed_call(q, k, v, [0, 110], 4, 2, 64, 110), want, 2 * bound, floor=2.0 ** -149)


@pytest.mark.parametrize("low,high", [(-100, 20), (-126, -100), (-40, 40), (-3, 3), (100, 126)])
@pytest.mark.parametrize("seen,new", [([0, 30], [70, 40]), ([3000], [50])])
def test_values_of_many_magnitudes(low, high, seen, new):
    rng = np.random.default_rng(high - low)
    x = Paged(rng, seen, new, 16, 4, 2, 64, "f32", make=lambda name, r, total: rng.uniform(-1, 1, (total, 2, 64)) * (
        3 if name == "k" else np.exp2(rng.integers(low, high + 1, (total, 1, 1)))))
    compare_many(x)


@pytest.mark.parametrize("power", [-116, -60, -30, -12, -8, 0, 30])
@pytest.mark.parametrize("zeros", [[0], [5, 6, 40], list(range(32)), list(range(64, 99))])
@pytest.mark.parametrize("score", [0, 12])
def test_rows_of_zeros_beside_small_values(power, zeros, score):
    """A value row of zeros adds nothing to a row's sum, so the others keep their bits, also where it has the largest weight."""
    rng = np.random.default_rng(len(zeros) + score)

    def make(name, r, total):
        if name == "k":
            return keys_below(rng, total, zeros, [score] * len(zeros))
        v = rng.standard_normal((total, 2, 64)) * 2.0 ** power
        v[zeros] = 0
        return v

    x = Paged(rng, [100], [70], 16, 4, 2, 64, "f32", make=make)
    queries(x)
    compare_many(x)
