"""Frequencies as 64-bit fractions of a turn, against exact fractions."""
import math

import numpy as np
import pytest

from _turns import off
from laya_rust_b200 import engine as E
from laya_rust_b200 import ops


def frequencies():
    for rot in (2, 64, 128, 512):
        for base in (1e4, 1.6e5, 5e5):
            yield from ops.rope_freqs(base, rot)[0]
            yield from ops.rope_freqs(base, rot, ops.RopeScaling(ops.ROPE_LINEAR, 8.0))[0]
    yield from np.exp(np.random.default_rng(0).uniform(math.log(1e-18), math.log(2.0 ** 20), 2000))
    yield from (2.0 ** 20, 2 * math.pi, 1e-17, 3e-16, 1e-30, 5e-324, 0.0)


def test_negative_frequencies_are_the_mirror():
    """The same error as their positive twins, which is under one 2^-64 of a turn."""
    for f in frequencies():
        assert (ops.rope_turns(float(f)) + ops.rope_turns(-float(f))) % 2 ** 64 == 0, f
        assert off(-f, ops.rope_turns(-float(f))) < 1, f


@pytest.mark.parametrize("f", [float("nan"), float("inf"), -float("inf"), 2.0 ** 20 + 1, -(2.0 ** 20) - 1])
def test_bad_frequencies_are_refused(f):
    with pytest.raises(E.LayaError, match="frequency") as ei:
        ops.rope_turns(f)
    assert ei.value.code == E.LAYA_E_INVALID


def test_null_argument():
    assert ops.lib().laya_rope_turns(1.0, None) == E.LAYA_E_INVALID


def test_the_fraction_is_rounded_once():
    """Half a 2^-64 of a turn.  Beyond that the constant's two doubles leave 2^-107 of
    it, at most 2^20 / (2 pi) turns * 2^64 * 2^-107 = 2^-26 units, and the low
    parts, up to 2^27 units, their own rounding of 2^-26."""
    worst = max((off(s * f, ops.rope_turns(s * float(f))), s * f) for f in frequencies() for s in (1, -1))
    assert worst[0] <= 0.5 + 2.0 ** -24, worst
