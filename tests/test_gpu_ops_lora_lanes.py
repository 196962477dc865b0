"""Warps whose 32 rows have many adapters: the lanes of one warp store different
entries, then load from tensor memory together again.  On every kernel that does
so, with inputs whose sums are exact (see _lora_rank)."""
import pytest
import torch

import _lora_rank as L
from test_gpu_ops_lora import BOTH, DT, Case

pytestmark = pytest.mark.gpu

# rows (one a segment), adapters, rank, in, out
SHAPES = [(12000, 8, 16, 256, 512),     # items by themselves, 8 entries each
          (12000, 3, 40, 72, 264),
          (2600, 20, 16, 1024, 1024),   # items in a cluster
          (128, 8, 16, 64, 1024),       # a CTA by itself, x on the M side against A
          (100, 8, 16, 64, 1024), (100, 8, 16, 1024, 512), (60, 3, 20, 512, 512), (90, 4, 16, 1024, 3072)]


@BOTH
@pytest.mark.parametrize("rows,ads,rank,inn,out", SHAPES)
def test_rows_of_a_warp_with_different_adapters(type, rows, ads, rank, inn, out):
    slots = [(i * 7 + i // 32) % (ads + 1) - 1 for i in range(rows)]     # one in ads + 1 without
    ranks = [rank - (i % 3) for i in range(ads)]
    ranks[0] = rank
    c = Case(type, [1] * rows, slots, ranks, inn, out)
    x, w, c.a, c.b, c.scale, owner = L.exact_inputs(DT[type], [1] * rows, slots, ranks, inn, out, rows, "cuda")
    c.xb[:c.m, :inn], c.wb[:, :inn] = x, w
    for i in range(ads):
        c.put(i)
    want, part = L.definition(x, w, c.a, c.b, c.scale, owner)
    lim = L.rank_limit(DT[type], want, part, 1.0)
    c.run()
    c.plan.status()
    assert bool(((c.y().double() - want).abs() <= lim).all())
    first = c.y().clone()
    for _ in range(5):
        c.run()
        assert torch.equal(c.y(), first)
