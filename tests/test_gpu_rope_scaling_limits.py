"""laya_set_rope_scaling on a model whose own frequencies are broken: refused before
anything changes, like bad parameters."""
import numpy as np
import pytest

from laya_rust_b200 import arch, modelgen, ops, workloads
from laya_rust_b200 import engine as E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -2.0**22])
def test_frequencies_no_table_can_be_made_from_are_refused(bad):
    eng = E.Engine(modelgen.cached_model(seed=0), device=0)
    try:
        req = workloads.long_state(seed=6)
        base = eng.forward(req)
        f = np.ones(32, np.float32)
        f[7] = bad
        eng.upload_f32(arch.ROPE_FREQ_SLIDING, f)
        with pytest.raises(E.LayaError, match="frequency") as ei:
            ops.set_rope_scaling(eng, None, ops.RopeScaling(ops.ROPE_LINEAR, 2.0))
        assert ei.value.code == E.LAYA_E_INVALID
        assert np.array_equal(eng.forward(req).logits, base.logits)
    finally:
        eng.close()


def test_the_limit_holds_for_the_stretched_frequency():
    """-2^21 / 2 is -2^20, the largest that is taken."""
    eng = E.Engine(modelgen.cached_model(seed=0), device=0)
    try:
        f = np.ones(32, np.float32)
        f[7] = -2.0**21
        eng.upload_f32(arch.ROPE_FREQ_SLIDING, f)
        ops.set_rope_scaling(eng, None, ops.RopeScaling(ops.ROPE_LINEAR, 2.0))
        assert np.isfinite(eng.forward(workloads.long_state(seed=6)).logits).all()
        with pytest.raises(E.LayaError, match="frequency"):
            ops.set_rope_scaling(eng, None, ops.RopeScaling(ops.ROPE_LINEAR, 1.5))
    finally:
        eng.close()
