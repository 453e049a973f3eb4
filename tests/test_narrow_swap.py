"""Buffers of narrow types change places with their own kind only: in another's place their elements would be counted by another size."""
import numpy as np
import pytest
import torch

from smallframework_b200 import interface as S

CPU = dict(device="cpu")


def kinds():
    return [S.FloatBuffer(8, **CPU), S.QUInt8Buffer(8, **CPU), S.BFloat16Buffer(8, **CPU), S.HalfBuffer(8, **CPU), S.Float8Buffer(1, 8, **CPU)]


@pytest.mark.parametrize("a", range(5))
@pytest.mark.parametrize("b", range(2, 5))
def test_other_kinds_are_refused(a, b):
    if a == b:
        return
    x, y = kinds()[a], kinds()[b]
    tx, ty = x.t, y.t
    for one, two in ((x, y), (y, x)):
        with pytest.raises(ValueError, match="swap"):
            one.swap(two)
    assert x.t is tx and y.t is ty and x.t.dtype == type(x).dtype and y.t.dtype == type(y).dtype


def test_the_same_kind_changes_all_that_it_has():
    a = S.Float8Buffer(1, 4, data=np.uint8([0x38] * 4), scales=np.float32([2]), **CPU)
    b = S.Float8Buffer(130, 16, 128, data=torch.full((130, 16), 0xb8, dtype=torch.uint8), **CPU)
    a.swap(b)
    assert (a.rows, a.columns, a.block_rows, b.rows, b.columns, b.block_rows) == (130, 16, 128, 1, 4, 1)
    assert (a.dequantized() == -1).all() and (b.dequantized() == 2).all()
    x, y = S.FloatBuffer(data=np.float32([1]), **CPU), S.FloatBuffer(data=np.float32([2, 3]), **CPU)
    x.swap(y)
    assert x.numpy().tolist() == [2, 3] and y.numpy().tolist() == [1]
