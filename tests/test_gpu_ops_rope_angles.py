"""Angles of laya_rope at any 32-bit position and frequency, against exact fractions.

x is (1, 0) in every pair, so the output is the cosine and the sine themselves.
The angle is off by at most 2^-32 of a turn (1.5e-9), the reduced argument by half a
step (pi / 4 * 2^-24 = 4.7e-8), sincospi by two (1.2e-7), the factor rounds once
(6e-8): under 2.3e-7."""
import numpy as np
import pytest
import torch

from _turns import cos_sin
from laya_rust_b200 import ops
from test_gpu_ops_rope import rt, stream

pytestmark = pytest.mark.gpu

POS = [0, 1, -1, 2**31 - 1, -2**31, -2**31 + 1, 2**30 + 7, 123456789, -987654321, 1 << 20]


@pytest.mark.parametrize("layout", [ops.ROPE_HALF, ops.ROPE_INTERLEAVED])
@pytest.mark.parametrize("sign", [1, -1])
def test_positions_and_frequencies_of_both_signs(layout, sign):
    freqs = sign * np.concatenate([ops.rope_freqs(b, 64)[0] for b in (1e4, 5e5)] + [[1e-6, 1e-9, 1e-17, 3e-16, 0.0, 2.0**20, 12.5, 1e5]])
    n = len(freqs)
    pos = torch.tensor(POS, dtype=torch.int32, device="cuda")
    x = torch.zeros(len(POS), 1, 2 * n, device="cuda")
    c, s = (slice(0, n), slice(n, None)) if layout == ops.ROPE_HALF else (slice(0, None, 2), slice(1, None, 2))
    x[..., c] = 1.0
    out = torch.empty_like(x)
    ops.rope(ops.RopeSpec(ops.F32, 2 * n, 2 * n, freqs, layout), [rt(x, out)], len(POS), pos=pos.data_ptr(), stream=stream())
    want = np.array([[cos_sin(p, f) for f in freqs] for p in POS])
    got = out[:, 0].double().cpu().numpy()
    for k, part in ((0, c), (1, s)):
        err = np.abs(got[:, part] - want[..., k])
        assert err.max() <= 2.3e-7, (float(err.max()), np.unravel_index(err.argmax(), err.shape))
