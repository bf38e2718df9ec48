"""Which parts of a unit that several work ranges share are merged, through the
library's host view of it (``pcp_chunk_cut_parts``, the code the kernel runs):
all of them up to the one that ends the unit, or none when a range among them
gave up -- and never one behind the last range."""

from __future__ import annotations

import ctypes
import random

import pytest

from aws_training_study_b200 import _capi


def _parts(states, failed, g):
    out = ctypes.c_int32(-1)
    _capi.check(_capi.lib().pcp_chunk_cut_parts(_capi.int32_array(states), _capi.int32_array(failed), len(states), g,
                                                ctypes.byref(out)))
    return out.value


def _plain(states, failed, g):
    if failed[g]:
        return 0
    for i in range(g + 1, len(states)):
        if failed[i] or states[i] == 0:
            return 0
        if states[i] == 2:
            return i - g + 1
    return 0


@pytest.mark.parametrize("ranges", [1, 2, 31, 32, 33, 34, 74, 148])
def test_a_unit_over_all_ranges(ranges):
    states = [0] + [1] * (ranges - 2) + [2] if ranges > 1 else [0]
    ok = [0] * ranges
    assert _parts(states, ok, 0) == (ranges if ranges > 1 else 0)
    # the range that ends the unit gave up and left no record: nothing is read
    # past the last range
    assert _parts(states[:-1] + [0], ok, 0) == 0
    for bad in {0, ranges // 2, ranges - 1}:
        assert _parts(states, [int(i == bad) for i in range(ranges)], 0) == 0


def test_units_behind_one_another():
    rng = random.Random(0)
    for _ in range(300):
        n = rng.randrange(1, 149)
        states = [rng.choice([0, 1, 1, 1, 1, 1, 2]) for _ in range(n)]
        failed = [int(rng.random() < 0.02) for _ in range(n)]
        for g in range(n):
            got = _parts(states, failed, g)
            assert got == _plain(states, failed, g) and g + got <= n


def test_refusals():
    lib, one = _capi.lib(), _capi.int32_array([0])
    out = ctypes.c_int32()
    for args in ((None, one, 1, 0), (one, None, 1, 0), (one, one, 0, 0), (one, one, 1, 1), (one, one, 1, -1)):
        assert lib.pcp_chunk_cut_parts(*args, ctypes.byref(out)) == 1
    assert lib.pcp_chunk_cut_parts(one, one, 1, 0, None) == 1
