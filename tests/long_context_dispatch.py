"""Which kernel the attention calls over an 8-bit cache and in a window take, from the sizes: AttendManyRows of
accelep_amd/csrc/attend_common.h, with its numbers read there, so that a test knows which kernel it looks at."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np

_HEADER = (Path(__file__).resolve().parent.parent / "accelep_amd" / "csrc" / "attend_common.h").read_text()


def _pairs(name):
    mi, = re.findall(rf"constexpr int64_t {name} = (\d+) << 20;", _HEADER)
    return int(mi) << 20


Q8, F32 = _pairs("kPromptPairsQ8"), _pairs("kPromptPairsF32")  # pairs of rows and keys for the kernel of many rows


def takes_many_rows(pairs, seq, position, heads, kv_heads, window=0, sinks=0):
    group, end = heads // kv_heads, position + seq
    rows = seq * group
    whole = window == 0 or window >= end
    keys = end if whole else min(end, window + min(seq, (14 + group) // group + 1) + 32)
    steps = -(-keys // 32) + (0 if whole else -(-min(sinks, end) // 32))
    return rows > 16 and -(-rows // 16) * 16 >= -(-pairs // (steps * 32 * kv_heads))


def many(q, copies, pairs, position, kv_heads, window=0, sinks=0):
    """`copies` of each query head: one for the kernel of few rows, more for the one of many."""
    out = np.repeat(q, copies, axis=1)
    assert takes_many_rows(pairs, q.shape[0], position, out.shape[1], kv_heads, window, sinks) == (copies > 1)
    return out
