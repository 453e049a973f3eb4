"""Strides that rows do not fit into are refused before any buffer is looked at: 0 means packed to the library, whose rows a buffer of one row does not hold."""
import pytest

from smallframework_b200 import interface as S


@pytest.mark.parametrize("stride", [0, -256, 255, 1 << 63])
def test_rows_do_not_overlap(stride):
    cpu = dict(device="cpu")
    x, w = S.Float8Buffer(3, 256, **cpu), S.Float8Buffer(256, 256, 128, **cpu)
    one = S.FloatBuffer(256, **cpu)
    with pytest.raises(ValueError, match="apart"):
        S.QuantizeBlocks(3, 256, one, x, input_stride=stride)
    with pytest.raises(ValueError, match="apart"):
        S.Dense_Bias_Activation(256, 256, x, w, None, one, batch=3, output_stride=stride)
    with pytest.raises(ValueError, match="apart"):
        S.LogProbabilities(3, 256, one, None, None, S.FloatBuffer(3, **cpu), row_stride=stride)
