"""Rotary operator, host side: frequencies against their formulas in 64 bits
and every refusal laya_rope makes before it touches a device."""
import math
import os
import re

import numpy as np
import pytest

from laya_rust_b200 import engine as E
from laya_rust_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_operator_the_header_declares():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "laya_ops.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(laya_[a-z0-9_]+)\s*\(", text))
    assert {"laya_rope", "laya_rope_freqs", "laya_set_rope_scaling"} <= names
    missing = [n for n in names if not hasattr(ops.lib(), n)]
    assert not missing, missing


@pytest.mark.parametrize("rot", [2, 4, 20, 64, 128, 512])
@pytest.mark.parametrize("base", [10000.0, 160000.0])
def test_frequencies(rot, base):
    f, m = ops.rope_freqs(base, rot)
    assert m == 1.0
    # pow in 64 bits: a few units in the last place
    np.testing.assert_allclose(f, [math.exp(-2 * j / rot * math.log(base)) for j in range(rot // 2)], rtol=1e-14)


def test_linear_and_base_stretch():
    f0, _ = ops.rope_freqs(10000.0, 64)
    f, m = ops.rope_freqs(10000.0, 64, ops.RopeScaling(ops.ROPE_LINEAR, 4.0))
    np.testing.assert_allclose(f, f0 / 4, rtol=1e-15)
    assert m == 1.0
    f, m = ops.rope_freqs(10000.0, 64, ops.RopeScaling(ops.ROPE_BASE, 4.0))
    assert f[0] == f0[0] and math.isclose(f[-1], f0[-1] / 4, rel_tol=1e-14)
    np.testing.assert_allclose(f, (10000.0 * 4 ** (64 / 62)) ** (-2 * np.arange(32) / 64), rtol=1e-13)
    f, m = ops.rope_freqs(10000.0, 64, ops.RopeScaling(ops.ROPE_LINEAR, 1.0, attn=1.5))
    assert np.array_equal(f, f0) and m == 1.5


def test_stretch_by_parts():
    L, lo, hi, s = 512.0, 1.0, 32.0, 8.0
    f0, _ = ops.rope_freqs(10000.0, 64)
    f, m = ops.rope_freqs(10000.0, 64, ops.RopeScaling(ops.ROPE_PARTS, s, L, lo, hi))
    turns = L * f0 / (2 * math.pi)
    g = np.clip((turns - lo) / (hi - lo), 0, 1)
    np.testing.assert_allclose(f, f0 * g + f0 / s * (1 - g), rtol=1e-14)
    assert g.min() == 0 and g.max() == 1      # both ends are in play
    assert m == np.float32(0.1 * math.log(s) + 1)


@pytest.mark.parametrize("base,rot,scaling", [
    (10000.0, 3, None), (10000.0, 0, None), (10000.0, 514, None), (0.0, 64, None), (float("nan"), 64, None),
    (10000.0, 64, ops.RopeScaling(7, 2.0)), (10000.0, 64, ops.RopeScaling(ops.ROPE_LINEAR, 0.5)),
    (10000.0, 64, ops.RopeScaling(ops.ROPE_LINEAR, float("inf"))), (10000.0, 2, ops.RopeScaling(ops.ROPE_BASE, 2.0)),
    (10000.0, 64, ops.RopeScaling(ops.ROPE_PARTS, 2.0)), (10000.0, 64, ops.RopeScaling(ops.ROPE_PARTS, 2.0, 512.0, 4.0, 4.0)),
    (10000.0, 64, ops.RopeScaling(ops.ROPE_LINEAR, 2.0, attn=-1.0)),
    (10000.0, 64, ops.RopeScaling(ops.ROPE_NONE, 1.0, attn=float("nan")))])
def test_bad_frequencies_are_refused(base, rot, scaling):
    with pytest.raises(E.LayaError) as ei:
        ops.rope_freqs(base, rot, scaling)
    assert ei.value.code == E.LAYA_E_INVALID


FAKE = 1 << 20  # never read: every call below is refused before its first device access


def tensor(**kw):
    d = dict(x=FAKE, out=2 * FAKE, heads=4, x_token=256, x_head=64, out_token=256, out_head=64)
    d.update(kw)
    return ops.RopeTensor(**d)


def spec(type=ops.F16, dim=64, rot=64, layout=ops.ROPE_HALF, mscale=1.0, freqs=None):
    return ops.RopeSpec(type, dim, rot, np.ones(max(rot, 0) // 2) if freqs is None else freqs, layout, mscale=mscale)


@pytest.mark.parametrize("why,call", [
    ("type", lambda: ops.rope(spec(type=9), [tensor()], 4)),
    ("layout", lambda: ops.rope(spec(layout=2), [tensor()], 4)),
    ("dim", lambda: ops.rope(spec(dim=514, rot=64), [tensor()], 4)),
    ("rot", lambda: ops.rope(spec(rot=66), [tensor()], 4)),
    ("rot", lambda: ops.rope(spec(rot=33), [tensor()], 4)),
    ("mscale", lambda: ops.rope(spec(mscale=float("inf")), [tensor()], 4)),
    ("frequency", lambda: ops.rope(spec(freqs=np.full(32, np.nan)), [tensor()], 4)),
    ("frequency", lambda: ops.rope(spec(freqs=np.full(32, 2.0e6)), [tensor()], 4)),
    ("pos", lambda: ops.rope(spec(), [tensor()], 4, pos=FAKE + 2)),
    ("65535", lambda: ops.rope(spec(), [tensor(heads=40000, out_head=64, out_token=40000 * 64)] * 2, 4)),
    ("1 to 4", lambda: ops.rope(spec(), [], 4)),
    ("1 to 4", lambda: ops.rope(spec(), [tensor()] * 5, 4)),
    ("tokens", lambda: ops.rope(spec(), [tensor()], -1)),
    ("32 bits", lambda: ops.rope(spec(), [tensor()], 4, pos0=2**31 - 3)),
    ("heads", lambda: ops.rope(spec(), [tensor(heads=-1)], 4)),
    ("null", lambda: ops.rope(spec(), [tensor(x=0)], 4)),
    ("aligned", lambda: ops.rope(spec(), [tensor(x=FAKE + 1)], 4)),
    ("negative", lambda: ops.rope(spec(), [tensor(x_head=-64)], 4)),
    ("too large", lambda: ops.rope(spec(), [tensor(x_token=2**41)], 4)),
    ("overlap", lambda: ops.rope(spec(), [tensor(out_head=32)], 4)),
    ("overlap", lambda: ops.rope(spec(), [tensor(out_token=255)], 4)),
    ("overlap", lambda: ops.rope(spec(), [tensor(out_token=0)], 4)),
    ("overlap", lambda: ops.rope(spec(), [tensor(heads=1, out_token=63)], 4)),
    ("overlap", lambda: ops.rope(spec(), [tensor(out_head=4 * 64 - 1, out_token=64)], 4)),
    ("equal strides", lambda: ops.rope(spec(), [tensor(out=FAKE, out_token=512)], 4))])
def test_bad_calls_are_refused(why, call):
    with pytest.raises(E.LayaError, match=why) as ei:
        call()
    assert ei.value.code == E.LAYA_E_INVALID


def test_nothing_to_do_is_no_error():
    ops.rope(spec(), [tensor()], 0)
    ops.rope(spec(), [tensor(heads=0)], 4)


def test_null_arguments():
    assert ops.lib().laya_rope(0, None, None, 1, 1, None, 0, None) == E.LAYA_E_INVALID
    assert ops.lib().laya_rope_freqs(1e4, 64, None, None, None) == E.LAYA_E_INVALID
    assert ops.lib().laya_set_rope_scaling(None, None, None) == E.LAYA_E_INVALID
