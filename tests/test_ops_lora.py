"""Low-rank adapters, host side: the plan of a batch against a plain
restatement, and every refusal made before a device is touched."""
import numpy as np
import pytest

from laya_rust_b200 import engine as E
from laya_rust_b200 import ops


def plain_layout(rows, slots, ranks):
    owner = [s for r, s in zip(rows, slots) for _ in range(r)]
    off, chunks = [0], []
    for b in range(0, len(owner), 256):
        seen = []
        for s in owner[b:b + 256]:
            if s >= 0 and s not in seen:
                seen.append(s)
        chunks += [(s, c) for s in seen for c in range((ranks[s] + 15) // 16)]
        off.append(len(chunks))
    return off, chunks


@pytest.mark.parametrize("rows,slots,ranks", [
    ([1], [0], [16]), ([1], [-1], [16]), ([0, 0], [0, -1], [4]), ([], [], [4]), ([256], [0], [17]), ([257], [0], [1]),
    ([100, 0, 156, 1], [1, 0, 1, 0], [16, 256]), ([3] * 90, [i % 5 for i in range(90)], [1, 15, 16, 17, 33]),
    ([700, 20, 700], [2, -1, 0], [8, 0, 40]), ([1] * 300, [i for i in range(300)], [16] * 300)])
def test_layout(rows, slots, ranks):
    off, chunks = ops.lora_layout(rows, slots, ranks)
    want_off, want = plain_layout(rows, slots, ranks)
    assert off.tolist() == want_off and [tuple(c) for c in chunks.tolist()] == want


def test_layout_of_random_batches():
    rng = np.random.default_rng(0)
    for _ in range(50):
        n, k = int(rng.integers(1, 60)), int(rng.integers(1, 12))
        rows, slots, ranks = rng.integers(0, 90, n), rng.integers(-1, k, n), rng.integers(1, 257, k)
        off, chunks = ops.lora_layout(rows, slots, ranks)
        want_off, want = plain_layout(rows, slots, ranks)
        assert off.tolist() == want_off and [tuple(c) for c in chunks.tolist()] == want


@pytest.mark.parametrize("why,rows,slots,ranks", [
    ("negative", [-1], [0], [4]), ("out of range", [1], [1], [4]), ("out of range", [1], [-2], [4]),
    ("empty", [1], [0], [0]), ("rank", [1], [0], [257]), ("too many rows", [2**24, 1], [0, 0], [4]),
    ("too many rows", [2**31 - 1, 2**31 - 1], [0, 0], [4])])
def test_bad_segments_are_refused(why, rows, slots, ranks):
    with pytest.raises(E.LayaError, match=why) as ei:
        ops.lora_layout(rows, slots, ranks)
    assert ei.value.code == E.LAYA_E_INVALID


FAKE = 1 << 20  # never read: every call below is refused before its first device access


@pytest.mark.parametrize("why,kw", [
    ("null", dict(w=0)), ("type", dict(type=ops.F32)), ("in and out", dict(inn=0)), ("in and out", dict(out=1 << 21)),
    ("ldw", dict(ldw=56)), ("16 bytes", dict(ldw=65, inn=65)), ("16 bytes", dict(w=FAKE + 8)),
    ("bias", dict(bias=FAKE + 2)), ("slots", dict(slots=0)), ("slots", dict(slots=4097)), ("max_rank", dict(max_rank=0)),
    ("max_rank", dict(max_rank=257)), ("too large", dict(slots=4096, max_rank=256, out=1 << 16))])
def test_bad_projections_are_refused(why, kw):
    d = dict(type=ops.F16, inn=64, out=128, w=FAKE, ldw=64)
    d.update(kw)
    with pytest.raises(E.LayaError, match=why) as ei:
        ops.Lora(**d)
    assert ei.value.code == E.LAYA_E_INVALID


def test_null_handles():
    L = ops.lib()
    assert L.laya_lora_create(0, 0, 64, 64, FAKE, 64, None, 1, 16, None) == E.LAYA_E_INVALID
    assert L.laya_lora_set(None, 0, 1, None, None, 0, 1.0) == E.LAYA_E_INVALID
    assert L.laya_lora_clear(None, 0) == E.LAYA_E_INVALID
    assert L.laya_lora_plan_create(None, None, None, 0, None) == E.LAYA_E_INVALID
    assert L.laya_lora_run(None, None, None, 0, None, 0, None) == E.LAYA_E_INVALID
    assert L.laya_lora_status(None) == E.LAYA_E_INVALID
    L.laya_lora_destroy(None)
    L.laya_lora_plan_destroy(None)
    assert L.laya_adapters_create(None, 1, 16) == E.LAYA_E_INVALID
    assert L.laya_adapter_create(None, 0, 16, 1.0) == E.LAYA_E_INVALID
    assert L.laya_adapter_upload(None, 0, b"x", None, None, 0) == E.LAYA_E_INVALID
    assert L.laya_adapter_drop(None, 0) == E.LAYA_E_INVALID
    assert L.laya_forward_adapted(None, None, None, None, None) == E.LAYA_E_INVALID
    assert L.laya_plan_create_adapted(None, None, None, None) == E.LAYA_E_INVALID
