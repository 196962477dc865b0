"""Every device-side wait of the adapter projection is bounded.  The next run of a
plan is made to wait, 1 ms long, for loads that a barrier holds back or for sums
that no thread block of the cluster sends.  It must return, laya_lora_status must
report LAYA_E_DEVICE_TIMEOUT, and the next run must be right again."""
import pytest
import torch

from laya_rust_b200 import engine as E
from laya_rust_b200 import ops
from test_gpu_ops_lora import BOTH, Case

pytestmark = pytest.mark.gpu

# rows and slots, ranks, in, out, what can be made to wait
CASES = [([1], [0], [16], 1024, 3072, (1, 2)),                                    # one launch in clusters of 8
         ([60, 100], [0, 1], [16, 60], 2624, 1024, (1, 2)),                       # rank values apart
         ([100], [0], [16], 1024, 512, (1, 2)),
         ([100, 100], [0, 1], [64, 64], 64, 1024, (1,)),                          # a CTA by itself
         ([1] * 48, list(range(48)), [16] * 48, 1024, 1024, (1, 2)),              # pairs, then clusters
         ([24] * 70, [i % 20 for i in range(70)], [128] * 20, 1024, 1024, (0, 1, 2)),   # items in clusters
         ([1500, 1500], [0, 1], [16, 60], 1024, 3072, (0, 1)),                    # the GEMM
         ([3000, 3000, 6600], [0, 1, -1], [16, 16], 256, 512, (0, 1))]             # items by themselves


@BOTH
@pytest.mark.parametrize("case", CASES, ids=[f"{sum(c[0])}x{c[3]}x{c[4]}-{len(c[2])}" for c in CASES])
def test_an_expired_wait_is_reported_and_the_plan_recovers(type, case):
    rows, slots, ranks, inn, out, kinds = case
    c = Case(type, rows, slots, ranks, inn, out, bias=True)
    c.run()
    c.check()
    first = c.y().clone()
    for kind in kinds:
        c.plan.test_timeout_next(kind, 1_000_000)
        c.run()
        with pytest.raises(E.LayaError, match="wait expired") as ei:
            c.plan.status()
        assert ei.value.code == E.LAYA_E_DEVICE_TIMEOUT
        # rows behind the last segment and columns up to the pitch stay even then
        assert bool((c.yb[c.m:] == 7.0).all()) and bool((c.yb[:, c.out:] == 7.0).all())
        c.yb.fill_(7.0)
        c.run()
        c.check()
        assert torch.equal(c.y(), first)


def test_bad_arguments_are_refused():
    c = Case(ops.F16, [4], [0], [8], 64, 64)
    for kind, lim in ((-1, 1000), (3, 1000), (1, 0), (1, 3_000_000_000), (0, 1000)):
        with pytest.raises(E.LayaError) as ei:
            c.plan.test_timeout_next(kind, lim)
        assert ei.value.code == E.LAYA_E_INVALID
    c.run()
    c.check()
    assert ops.lib().laya_lora_test_timeout_next(None, 1, 1000) == E.LAYA_E_INVALID
