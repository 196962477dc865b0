"""laya_lora_* on the B200 against the formula in 64 bits.

Tolerance, per element of y.  Let S1 = sum |x W| + |bias| and S2 = scale *
sum_j (sum_k |x A_j|) |B_j|, the sums of magnitudes.  Products of 16-bit values
are exact in f32, and an f32 sum of n terms in any order is off by at most
n 2^-24 of the sum of magnitudes.  The tensor core adds the products of one
step (16 terms) after aligning them to the largest, keeping at least 2 bits
below an f32 mantissa's, and truncates: under 2^-22 of the magnitudes for each
of its in / 16 steps, so 2^-22 (in / 16 + 1) in all, which is no more than
(in + 16) 2^-24 for in >= 3 * 16 and covered by the bound below with the
factor 4.  Between the products scale x A^T is rounded to one f16 (off by at
most eps, half a step, of each value) or to a pair of bf16 (2 eps^2), and the
scale rounds once.  So
  |error| <= 4 (in + rank + 32) 2^-24 (S1 + S2) + r S2,  r = eps (f16), 2 eps^2 (bf16)
and y rounds by at most eps |y| (2^-25 for f16 values below its normal range;
rank values below f16's normal range add 2^-25 sum_j |B_j|).
"""
import numpy as np
import pytest
import torch

from laya_rust_b200 import engine as E
from laya_rust_b200 import ops

pytestmark = pytest.mark.gpu
DT = {ops.F16: torch.float16, ops.BF16: torch.bfloat16}


def up8(n):
    return (n + 7) // 8 * 8


class Case:
    def __init__(self, type, rows, slots, ranks, inn, out, bias=False, seed=0, pitch=0, max_rank=None, fill=float("nan"),
                 a_std=None):
        dt = DT[type]
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.type, self.rows, self.slots, self.inn, self.out = type, rows, slots, inn, out
        self.m = m = int(sum(rows))
        ldx, ldy = up8(inn) + pitch, up8(out) + pitch
        # what lies between the columns and the pitch must not be read as a value
        self.xb = torch.full((m + 3, ldx), fill, device="cuda", dtype=dt)
        self.xb[:m, :inn] = rnd(m, inn).to(dt)
        self.wb = torch.full((out, up8(inn) + pitch), fill, device="cuda", dtype=dt)
        self.wb[:, :inn] = (rnd(out, inn) * 0.05).to(dt)
        self.a = [(rnd(r, inn) * (a_std or inn ** -0.5)).to(dt) for r in ranks]
        self.b = [(rnd(out, r) * 0.1).to(dt) for r in ranks]
        self.scale = [1.5 + 0.25 * i for i in range(len(ranks))]
        self.bias = rnd(out) if bias else None
        self.yb = torch.full((m + 3, ldy), 7.0, device="cuda", dtype=dt)
        self.lora = ops.Lora(type, inn, out, self.wb.data_ptr(), self.wb.stride(0),
                             self.bias.data_ptr() if bias else 0, slots=max(1, len(ranks)),
                             max_rank=max_rank or max([1, *ranks]))
        for i in range(len(ranks)):
            self.put(i)
        self.plan = self.lora.plan(rows, slots)

    def put(self, i):
        self.lora.set(i, self.a[i].float().cpu().numpy(), self.b[i].float().cpu().numpy(), self.scale[i])

    def run(self, stream=None):
        s = stream or torch.cuda.current_stream()
        self.lora.run(self.plan, self.xb.data_ptr(), self.xb.stride(0), self.yb.data_ptr(), self.yb.stride(0),
                      stream=s.cuda_stream)

    def y(self):
        return self.yb[:self.m, :self.out]

    def want(self):
        x, w = self.xb[:self.m, :self.inn].double(), self.wb[:, :self.inn].double()
        y, s1, s2 = x @ w.T, x.abs() @ w.abs().T, torch.zeros(self.m, self.out, device="cuda", dtype=torch.float64)
        tiny, rank = torch.zeros_like(s2), 0
        if self.bias is not None:
            y, s1 = y + self.bias.double(), s1 + self.bias.double().abs()
        row = 0
        for r, s in zip(self.rows, self.slots):
            if s >= 0 and r:
                a, b, sl = self.a[s].double(), self.b[s].double(), slice(row, row + r)
                y[sl] += self.scale[s] * (x[sl] @ a.T) @ b.T
                s2[sl] = self.scale[s] * (x[sl].abs() @ a.abs().T) @ b.abs().T
                tiny[sl] = b.abs().sum(1) * 2.0 ** -25 if self.type == ops.F16 else 0.0
                rank = max(rank, a.shape[0])
            row += r
        eps = torch.finfo(DT[self.type]).eps / 2
        between = eps if self.type == ops.F16 else 2 * eps * eps
        tol = 4 * (self.inn + rank + 32) * 2.0 ** -24 * (s1 + s2) + between * s2 + tiny
        return y, tol

    def check(self):
        self.plan.status()
        y, tol = self.want()
        eps = torch.finfo(DT[self.type]).eps / 2
        err = (self.y().double() - y).abs()
        lim = tol + eps * (y.abs() + tol) + (2.0 ** -25 if self.type == ops.F16 else 0.0)
        assert bool((err <= lim).all()), (float((err - lim).max()), (err > lim).nonzero()[:5].tolist())
        # rows behind the last segment and columns up to the pitch stay
        assert bool((self.yb[self.m:] == 7.0).all()) and bool((self.yb[:, self.out:] == 7.0).all())


BOTH = pytest.mark.parametrize("type", [ops.F16, ops.BF16])


@BOTH
@pytest.mark.parametrize("inn,out", [(64, 128), (1024, 1024), (1000, 1531), (1, 1), (8, 3), (65, 257), (130, 255),
                                     (2624, 1024), (63, 40)])
@pytest.mark.parametrize("rows", [1, 2, 7, 16, 17, 33])
def test_few_rows(type, inn, out, rows):
    c = Case(type, [rows], [0], [16], inn, out, seed=rows)
    c.run()
    c.check()


@BOTH
@pytest.mark.parametrize("inn,out", [(1024, 3072), (1000, 1531), (2624, 1024), (72, 264)])
@pytest.mark.parametrize("m", [40, 64, 65, 127, 128, 129, 179, 256, 257, 385, 600, 1357, 2300])
def test_more_rows(type, inn, out, m):
    cut = m // 3
    c = Case(type, [cut, 0, 1, m - cut - 1], [1, 0, -1, 0], [16, 11], inn, out, bias=True, seed=m)
    c.run()
    c.check()


@BOTH
@pytest.mark.parametrize("inn,out", [(1024, 1024), (1000, 1531), (200, 136)])
@pytest.mark.parametrize("lens,slots,ranks", [
    # row tiles with 0, 1, 4, 5, 8 and 9 adapter chunks, adapters that start in the middle of a tile
    ([64] * 10, [-1, 0, -1, 1, 1, -1, 0, -1, -1, 1], [16, 9]),
    ([100, 30, 30, 30, 30, 100, 300], [0, 1, 2, 3, -1, 0, 2], [16, 16, 32, 7]),
    ([130, 130, 130], [0, 1, 2], [128, 112, 5]),
    ([500, 14, 14, 14], [0, 1, 2, 3], [64, 33, 16, 1]),
    ([8] * 70, [i % 9 for i in range(70)], [16] * 9),
    ([700, 3, 600], [-1, 0, -1], [100])])
def test_tiles_with_few_and_many_adapters(type, inn, out, lens, slots, ranks):
    c = Case(type, lens, slots, ranks, inn, out, bias=True, seed=len(lens))
    c.run()
    c.check()


@BOTH
@pytest.mark.parametrize("out", [5, 263, 8])
def test_many_rows_and_few_columns(type, out):
    """More rows than the few-row kernel takes, outputs narrower than a tile."""
    c = Case(type, [3000, 1, 3200], [0, -1, 1], [16, 5], 72, out, bias=True)
    c.run()
    c.check()


@BOTH
def test_a_large_packed_batch(type):
    rng = np.random.default_rng(1)
    rows = rng.integers(24, 129, 64).tolist()
    slots = rng.integers(-1, 9, 64).tolist()
    c = Case(type, rows, slots, [16, 1, 40, 128, 7, 33, 64, 16, 200], 1024, 1100, bias=True)
    c.run()
    c.check()


@BOTH
@pytest.mark.parametrize("rank", [1, 15, 16, 17, 31, 48, 64, 129, 256])
@pytest.mark.parametrize("m", [5, 300])
def test_ranks(type, rank, m):
    c = Case(type, [m], [0], [rank], 320, 300, max_rank=256)
    c.run()
    c.check()


@BOTH
@pytest.mark.parametrize("n,inn,out", [(1, 1024, 1024), (3, 1024, 1024), (16, 512, 700), (48, 1024, 1024), (300, 256, 320)])
def test_single_rows_each_with_an_adapter_of_its_own(type, n, inn, out):
    c = Case(type, [1] * n, list(range(n)), [1 + (5 * i) % 40 for i in range(n)], inn, out)
    c.run()
    c.check()


@BOTH
@pytest.mark.parametrize("n,rows,ads,ranks,inn,out", [
    (130, 1, 130, [16], 1024, 300), (256, 1, 256, [1, 20], 200, 520), (384, 1, 384, [16], 264, 1024), (700, 1, 90, [33, 5], 130, 257),
    (513, 1, 513, [16], 72, 64), (40, 25, 16, [64, 9], 264, 520), (11, 100, 10, [128, 200], 136, 640), (90, 7, 45, [17, 3], 1000, 131),
    (1100, 2, 300, [16], 64, 128), (37, 3, 20, [40], 512, 1024)])
def test_more_adapters_than_a_launch_takes(type, n, rows, ads, ranks, inn, out):
    """Row tiles with lists of their own, some segments without an adapter, and the GEMM behind them."""
    slots = [i % ads if i % 11 != 5 else -1 for i in range(n)]
    c = Case(type, [rows] * n, slots, [ranks[i % len(ranks)] for i in range(ads)], inn, out, bias=True, seed=n)
    c.run()
    c.check()
    first = c.y().clone()
    c.run()
    c.check()
    assert torch.equal(c.y(), first)


def test_no_adapter_anywhere_and_no_rows():
    c = Case(ops.F16, [70, 0, 9], [-1, -1, -1], [], 512, 256)
    c.run()
    c.check()
    e = Case(ops.F16, [0, 0], [0, -1], [4], 512, 256)
    e.run()
    assert bool((e.yb == 7.0).all())


def test_the_same_slot_again_and_again():
    c = Case(ops.BF16, [1, 2, 3, 250, 1, 260], [0, 1, 0, 1, 1, 0], [16, 24], 256, 512)
    c.run()
    c.check()


@BOTH
@pytest.mark.parametrize("m", [3, 20, 200, 700])
def test_pitches_and_repeated_runs(type, m):
    c = Case(type, [m], [0], [16], 200, 136, pitch=24)
    c.run()
    first = c.y().clone()
    c.check()
    for _ in range(3):
        c.yb.fill_(7.0)
        c.run()
        assert torch.equal(c.y(), first)      # bit for bit
    c.check()


def far_rows(t, pitch):
    """The rows of t at a pitch that takes their offsets past 2^32 elements."""
    assert (t.shape[0] - 1) * pitch > 1 << 32
    buf = torch.empty((t.shape[0] - 1) * pitch + up8(t.shape[1]), device="cuda", dtype=t.dtype)
    v = buf.as_strided(t.shape, (pitch, 1))
    v.copy_(t)
    return v


@BOTH
@pytest.mark.parametrize("rows,slots,pitch", [
    ([1] * 20, list(range(20)), 1 << 28),      # a block per (row, chunk)
    ([200], [0], 1 << 25),                     # one launch
    ([700, 3, 700], [0, -1, 1], 3 << 20),      # row tiles
    ([3000, 1100], [1, 0], 1 << 20)])          # the GEMM
def test_offsets_past_32_bits(type, rows, slots, pitch):
    c = Case(type, rows, slots, [16] * (max(slots) + 1), 200, 139)
    c.xb = far_rows(c.xb[:c.m, :c.inn], pitch + 8)
    c.yb = far_rows(c.yb[:c.m, :c.out], pitch)
    c.run()
    c.check()
    del c
    torch.cuda.empty_cache()


@BOTH
@pytest.mark.parametrize("m", [6, 300])
def test_a_row_with_infinities_or_nan_reaches_no_other_row(type, m):
    """The rows of all adapters share a tile; one request's broken activations
    must not touch its neighbours."""
    rows = [m // 3, m // 3, m - 2 * (m // 3)]
    c = Case(type, rows, [0, 1, -1], [16, 20], 256, 256)
    c.run()
    clean = c.y().clone()
    bad = [0, m // 3 + 1, m - 1]
    for i, v in zip(bad, (float("nan"), float("inf"), float("-inf"))):
        c.xb[i, 100] = v
    c.run()
    c.plan.status()
    keep = torch.ones(m, dtype=torch.bool, device="cuda")
    keep[bad] = False
    assert torch.equal(c.y()[keep], clean[keep])
    assert not bool(torch.isfinite(c.y()[~keep]).any())


def test_an_adapter_changed_between_runs():
    c = Case(ops.F16, [30, 30], [0, 1], [16, 10], 256, 256, max_rank=32)
    c.run()
    c.a[1] = torch.randn(5, 256, device="cuda").half() * 0.05      # rank 5: still one chunk, the plan stays
    c.b[1] = torch.randn(256, 5, device="cuda").half() * 0.1
    c.scale[1] = -3.0
    c.put(1)
    c.run()
    # S2's scale enters by magnitude
    c.plan.status()
    y, tol = c.want()
    assert bool(((c.y().double() - y).abs() <= tol.abs() * 4 + 2.0 ** -11 * y.abs() * 1.01 + 2.0 ** -25).all())
    c.a[1], c.b[1] = torch.randn(20, 256, device="cuda").half(), torch.randn(256, 20, device="cuda").half()
    c.put(1)                                                        # two chunks now
    with pytest.raises(E.LayaError, match="make a new plan") as ei:
        c.run()
    assert ei.value.code == E.LAYA_E_STATE
    c.lora.clear(1)
    with pytest.raises(E.LayaError, match="make a new plan"):
        c.run()
    with pytest.raises(E.LayaError, match="empty"):
        c.lora.plan([1], [1])


@pytest.mark.parametrize("m", [2, 100, 700])
def test_another_stream_and_a_replayed_graph(m):
    c = Case(ops.BF16, [m - 1, 1], [0, 1], [16, 32], 512, 384)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c.run(s)
    s.synchronize()
    c.check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    c.xb[:m, :512] = torch.randn(m, 512, device="cuda").to(torch.bfloat16)
    c.yb.fill_(7.0)
    g.replay()
    torch.cuda.synchronize()
    c.check()
    # an adapter changed in place reaches the replays
    c.a[0], c.b[0] = c.a[0] * -2, torch.randn_like(c.b[0].float()).to(torch.bfloat16) * 0.1
    c.put(0)
    g.replay()
    torch.cuda.synchronize()
    c.check()


@pytest.mark.parametrize("m", [3, 200])
def test_two_plans_on_two_streams_at_once(m):
    a = Case(ops.F16, [m], [0], [16], 512, 512, seed=1)
    b = Case(ops.F16, [m + 50], [0], [16], 512, 512, seed=2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        a.run(s1)
        b.run(s2)
    torch.cuda.synchronize()
    a.check()
    b.check()


def test_bad_calls_are_refused():
    c = Case(ops.F16, [4], [0], [8], 64, 64)
    ok = dict(x=c.xb.data_ptr(), ldx=c.xb.stride(0), y=c.yb.data_ptr(), ldy=c.yb.stride(0))
    host = torch.zeros(4, 64, dtype=torch.float16).data_ptr()
    host += -host % 16
    for why, kw in (("null", dict(x=0)), ("null", dict(y=0)), ("ldx", dict(ldx=56)), ("ldy", dict(ldy=56)),
                    ("16 bytes", dict(ldx=65)), ("16 bytes", dict(y=ok["y"] + 2)), ("16 bytes", dict(x=ok["x"] + 8)),
                    ("apart", dict(y=ok["x"])), ("not a device address", dict(x=host)), ("not a device address", dict(y=host))):
        with pytest.raises(E.LayaError, match=why) as ei:
            c.lora.run(c.plan, **{**ok, **kw})
        assert ei.value.code == E.LAYA_E_INVALID
    other = Case(ops.F16, [4], [0], [8], 64, 64)
    with pytest.raises(E.LayaError, match="another projection"):
        other.lora.run(c.plan, **ok)
    a, b = np.zeros((8, 64), np.float32), np.zeros((64, 8), np.float32)
    for why, f in (("slot", lambda: c.lora.set(1, a, b)), ("rank", lambda: c.lora.set(0, np.zeros((9, 64)), np.zeros((64, 9)))),
                   ("scale", lambda: c.lora.set(0, a, b, float("nan"))),
                   ("not finite", lambda: c.lora.set(0, a + np.inf, b)), ("not finite", lambda: c.lora.set(0, a, b + 1e6)),
                   ("slot", lambda: c.lora.clear(-1)), ("slot", lambda: c.lora.plan([1], [1])),
                   ("not a device address", lambda: ops.Lora(ops.F16, 64, 64, host, 64)),
                   ("device", lambda: ops.Lora(ops.F16, 64, 64, c.wb.data_ptr(), 64, device=99))):
        with pytest.raises(E.LayaError, match=why) as ei:
            f()
        assert ei.value.code == E.LAYA_E_INVALID
    c.run()
    c.check()
