"""Refusals of the engine's adapters at limits that are no multiple of a chunk."""
import pytest

from laya_rust_b200 import engine as E
from laya_rust_b200 import modelgen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_rank", [1, 10, 17])
def test_a_rank_above_max_rank_is_refused(max_rank):
    eng = E.Engine(modelgen.cached_model(seed=0), device=0)
    try:
        eng.adapters_create(2, max_rank)
        eng.adapter_create(0, max_rank, 1.0)
        for rank in (0, max_rank + 1, (max_rank + 15) // 16 * 16, 257):
            if rank == max_rank:
                continue
            with pytest.raises(E.LayaError, match="rank must be 1..max_rank") as ei:
                eng.adapter_create(1, rank, 1.0)
            assert ei.value.code == E.LAYA_E_INVALID
        eng.adapters_create(1, 32)          # the limit is the newest call's
        eng.adapter_create(0, 32, 1.0)
    finally:
        eng.close()
