"""What the adapter projection keeps of u = scale x A^T between its two
products, on every path that has one: inputs with exact sums (see _lora_rank),
and the rms of the adapter's part alone."""
import pytest
import torch

import _lora_rank as L
from laya_rust_b200 import ops
from test_gpu_ops_lora import BOTH, DT, Case

pytestmark = pytest.mark.gpu

# one launch, one tile or several, joint and apart; pairs with lists; items in
# clusters and alone; 128- and 256-column GEMM tiles, halves
SHAPES = [([1], [0], [16], 1024, 3072), ([1], [0], [256], 1024, 520), ([179], [0], [32], 2624, 1024),
          ([100, 79], [1, 0], [16, 120], 1024, 1024), ([256], [0], [16], 1024, 3072), ([128], [0], [100], 512, 2048),
          ([1] * 48, list(range(48)), [16] * 48, 1024, 1024), ([1] * 300, list(range(300)), [16] * 300, 256, 320),
          ([500, 400, 457], [0, 1, 2], [11, 16, 40], 1000, 1531), ([20] * 70, [i % 9 for i in range(70)], [16] * 9, 1000, 1536),
          ([1500, 0, 1500], [0, 1, 2], [16, 8, 60], 1024, 3072), ([77] * 130, [i % 17 - 1 for i in range(130)], [16] * 16, 1024, 1200),
          ([9, 3000], [0, 1], [200, 5], 72, 263)]
IDS = [f"{sum(s[0])}x{s[3]}x{s[4]}-{len(s[2])}r{max(s[2])}" for s in SHAPES]


@BOTH
@pytest.mark.parametrize("rows,slots,ranks,inn,out", SHAPES, ids=IDS)
def test_nothing_of_the_rank_values_is_lost(type, rows, slots, ranks, inn, out):
    c = Case(type, rows, slots, ranks, inn, out)
    x, w, c.a, c.b, c.scale, owner = L.exact_inputs(DT[type], rows, slots, ranks, inn, out, len(rows), "cuda")
    c.xb[:c.m, :inn], c.wb[:, :inn] = x, w
    for i in range(len(ranks)):
        c.put(i)
    c.run()
    c.plan.status()
    want, part = L.definition(x, w, c.a, c.b, c.scale, owner)
    lim = L.rank_limit(DT[type], want, part, 1.0)     # a row of B has one value, at most 1
    err = (c.y().double() - want).abs()
    assert bool((err <= lim).all()), (float((err - lim).max()), (err > lim).nonzero()[:5].tolist())


@BOTH
@pytest.mark.parametrize("rows,slots,ranks,inn,out", SHAPES, ids=IDS)
def test_the_adapter_part_alone_is_rounded_once(type, rows, slots, ranks, inn, out):
    """W = 0.  y = round(y exact + d), and d has two parts: eps^2 of u's values, and
    the f32 sums, each of at most 2624 / 16 tensor-core steps that are off by
    less than 2^-23 of what they hold: under 2^-15.6 of y's rms.  Rounding y leaves
    eps / sqrt(3) times a mean of 0.72 over the binade, 2^-12.2 in f16, the
    smaller of the two.  The parts are uncorrelated, so d raises the rms by
    2^(2 (12.2 - 15.6)) / 2 = 0.45% at most; 2% leaves room for the sample.  u
    rounded once would raise it by about 40%."""
    c = Case(type, rows, slots, ranks, inn, out)
    c.wb[:, :inn] = 0
    c.run()
    c.plan.status()
    want, _ = c.want()
    has = torch.repeat_interleave(torch.tensor(slots, device="cuda"), torch.tensor(rows, device="cuda")) >= 0
    want, got = want[has], c.y()[has]
    rounded = L.rms(want.to(DT[type]).double() - want)
    assert L.rms(got.double() - want) <= 1.02 * rounded, L.rms(got.double() - want) / rounded
