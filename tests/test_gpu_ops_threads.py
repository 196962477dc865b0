"""Calls on one projection from several threads at once: each run has the whole
of the adapter that was set before it or after it, never a part of either."""
import threading

import pytest
import torch

from laya_rust_b200 import ops
from test_gpu_ops_lora import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [3, 64, 1500])
def test_an_adapter_set_while_another_thread_runs(m):
    c = Case(ops.F16, [m], [0], [16], 1024, 1024)
    sets = [(c.a[0].float().cpu().numpy() * f, c.b[0].float().cpu().numpy() * g, h) for f, g, h in ((1, 1, 1.0), (-2, 0.5, 3.0))]
    want = []
    for v in sets:
        c.lora.set(0, *v)
        c.run()
        want.append(c.y().clone())
    torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    stop, failed = threading.Event(), []

    def setter():
        try:
            for i in range(300):
                c.lora.set(0, *sets[i % 2])
        except Exception as e:
            failed.append(e)
        stop.set()

    t = threading.Thread(target=setter)
    st, mixed, n = torch.cuda.Stream(), torch.zeros((), device="cuda", dtype=torch.int64), 0
    torch.cuda.synchronize()
    t.start()
    with torch.cuda.stream(st):
        while not stop.is_set() or n < 100:
            c.run(st)
            mixed += ~((c.y() == want[0]).all() | (c.y() == want[1]).all())
            n += 1
    t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    assert int(mixed) == 0, f"{int(mixed)} of {n} runs had parts of two adapters"


def test_plans_runs_and_ranks_from_many_threads():
    """Every call is right or refused for what it says: an adapter that changed its
    rank (make a new plan)."""
    c = Case(ops.BF16, [40], [0], [16], 256, 256, max_rank=48)
    a, b = c.a[0].float().cpu().numpy(), c.b[0].float().cpu().numpy()
    wide = [v.repeat(3, axis=ax) for v, ax in ((a, 0), (b, 1))]      # rank 48: three times the part
    c.run()
    narrow = c.y().clone()
    c.lora.set(0, *wide, c.scale[0] / 3)                             # the same sum
    torch.cuda.synchronize()
    failed = []

    def worker(i):
        try:
            st = torch.cuda.Stream()
            y = torch.empty_like(c.yb)
            for k in range(40):
                if i == 0:
                    c.lora.set(0, *(wide if k % 2 else (a, b)), c.scale[0] / (3 if k % 2 else 1))
                    continue
                p = c.lora.plan([40], [0])
                try:
                    c.lora.run(p, c.xb.data_ptr(), c.xb.stride(0), y.data_ptr(), y.stride(0), stream=st.cuda_stream)
                except Exception as e:
                    assert "make a new plan" in str(e), e
                    continue
                finally:
                    p.status()
                    p.close()
                st.synchronize()
                # another order of the same sum: a step of bf16 (2^-7) of the largest value
                err = (y[:40, :256].float() - narrow.float()).abs().max()
                assert float(err) <= 2.0 ** -7 * float(narrow.float().abs().max()), float(err)
        except Exception as e:
            failed.append(e)

    ts = [threading.Thread(target=worker, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
