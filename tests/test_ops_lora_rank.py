"""The bounds that the GPU tests of the rank-space vector assert, on the CPU:
met by a value and its remainder, missed by everything shorter."""
import pytest
import torch

import _lora_rank as L

CASE = ([5, 0, 40, 3, 16], [0, 1, 2, -1, 1], [16, 40, 7])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("inn", [72, 1024, 2624])
def test_exact_inputs_tell_a_pair_from_less(dtype, inn):
    rows, slots, ranks = CASE
    x, w, a, b, scale, owner = L.exact_inputs(dtype, rows, slots, ranks, inn, 100, 1, "cpu")
    want, part = L.definition(x, w, a, b, scale, owner)
    # the cancellation is there: 0 in the columns of an adapter's own rank values
    j = torch.arange(100) % 40
    assert bool((want[owner == 1] == 0).all()) and bool((want[owner == 2][:, j < 7] == 0).all())
    assert bool((want[owner == -1] != 0).any())
    lim = L.rank_limit(dtype, want, part, 1.0)

    def passes(held):
        y, _ = L.definition(x, w, a, b, scale, owner, held)
        return bool(((y.to(dtype).double() - want).abs() <= lim).all())

    assert passes(lambda u: u) and passes(L.pair(dtype))
    for short in (L.one(dtype), L.bits(8), L.bits(11)):
        assert not passes(short)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("inn,rank", [(1024, 16), (2624, 40)])
def test_rms_of_the_adapter_part_tells_a_pair_from_less(dtype, inn, rank):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(200, inn, generator=g).to(dtype)
    a, b = (torch.randn(rank, inn, generator=g) * inn ** -0.5).to(dtype), (torch.randn(300, rank, generator=g) * 0.1).to(dtype)
    args = x, torch.zeros(300, inn), [a], [b], [1.5], torch.zeros(200, dtype=torch.long)
    want, _ = L.definition(*args)
    ratio = lambda held: L.rms(L.definition(*args, held)[0].to(dtype).double() - want) / L.rms(want.to(dtype).double() - want)
    assert ratio(L.pair(dtype)) < 1.02
    for short in (L.one(dtype), L.bits(8)):
        assert ratio(short) > 1.2
