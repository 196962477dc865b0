"""Numbers that the operators' bindings and checks must not turn into others."""
import numpy as np
import pytest

from laya_rust_b200 import engine as E
from laya_rust_b200 import ops

WRONG = [np.array([2**32]), np.array([2**31]), np.array([-2**31 - 1]), np.array([2**32 - 1], np.uint64), [2**40],
         np.array([0.5]), [1.0], np.array([True])]


@pytest.mark.parametrize("v", WRONG, ids=[str(i) for i in range(len(WRONG))])
def test_numbers_that_int32_cannot_hold_are_refused(v):
    one = type("Req", (), dict(n=1))
    for f in (lambda: ops.lora_layout(v, [0], [4]), lambda: ops.lora_layout([1], v, [4]),
              lambda: ops.lora_layout([1], [0], v), lambda: E._adapter_array(one, v)):
        with pytest.raises(ValueError, match="32 bits"):
            f()


def test_whole_numbers_of_any_width_are_taken():
    one = type("Req", (), dict(n=1))
    for t in (np.int8, np.uint8, np.int32, np.int64, np.uint64):
        off, chunks = ops.lora_layout(np.array([3], t), np.array([0], t), np.array([17], t))
        assert off.tolist() == [0, 2] and chunks.tolist() == [[0, 0], [0, 1]]
        assert E._adapter_array(one, np.array([5], t)).tolist() == [5]
    assert ops.lora_layout([], [], [4])[0].tolist() == [0]
    with pytest.raises(E.LayaError, match="too many rows"):
        ops.lora_layout([2**31 - 1], [-1], [])
