"""Limits of the rotary operator's numbers, checked before a device is touched."""
import numpy as np
import pytest

from laya_rust_b200 import engine as E
from laya_rust_b200 import ops


@pytest.mark.parametrize("kind", [ops.ROPE_NONE, ops.ROPE_LINEAR, ops.ROPE_BASE, ops.ROPE_PARTS])
def test_a_factor_beyond_32_bits_is_refused(kind):
    """attn becomes a 32-bit factor on cos and sin: an infinite one would fill the
    engine's tables with infinities and NaN."""
    for attn in (3.5e38, 1e300):
        with pytest.raises(E.LayaError, match="attn") as ei:
            ops.rope_freqs(10000.0, 64, ops.RopeScaling(kind, 2.0, 512.0, 1.0, 32.0, attn))
        assert ei.value.code == E.LAYA_E_INVALID
    _, m = ops.rope_freqs(10000.0, 64, ops.RopeScaling(kind, 2.0, 512.0, 1.0, 32.0, 3.4e38))
    assert m == np.float32(3.4e38)


def test_every_32_bit_start_is_taken():
    """tokens == 0 does nothing, after the checks."""
    spec, t = ops.RopeSpec(ops.F16, 64, 64, np.ones(32)), ops.RopeTensor(0, 0, 1, 64, 64, 64, 64)
    for pos0 in (-2**31, -1, 0, 2**31 - 1):
        ops.rope(spec, [t], 0, pos0=pos0)
    for pos0 in (-2**31 - 1, 2**31 + 1, 2**63 - 1, -2**63):
        with pytest.raises(E.LayaError, match="32 bits"):
            ops.rope(spec, [t], 0, pos0=pos0)
