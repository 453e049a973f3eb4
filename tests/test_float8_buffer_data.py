"""What a Float8Buffer is made from: bytes are codes wherever they come from, numbers of other types are refused, and codes without scales have scales of 1."""
import numpy as np
import pytest
import torch

from smallframework_b200 import interface as S

CODES, VALUES = [0x38, 0xb8, 0x7e, 0x01], [1.0, -1.0, 448.0, 2.0 ** -9]


@pytest.mark.parametrize("data", [np.uint8(CODES), torch.tensor(CODES, dtype=torch.uint8), torch.tensor(CODES, dtype=torch.uint8).view(torch.float8_e4m3fn),
                                  np.uint8([CODES]), torch.tensor([CODES], dtype=torch.uint8), torch.tensor(CODES, dtype=torch.uint8).repeat_interleave(2)[::2]],
                         ids=["numpy", "torch", "e4m3", "numpy matrix", "torch matrix", "torch stride"])
def test_bytes_are_codes(data):
    b = S.Float8Buffer(1, 4, data=data, scales=np.float32([2]), device="cpu")
    assert b.t.dtype == torch.float8_e4m3fn and b.t.shape == (4,)
    assert b.dequantized().tolist() == [[2 * v for v in VALUES]]


def test_bytes_of_a_tensor_are_not_copied():
    """Codes are looked at where they are, as those of a float8 tensor are."""
    codes = torch.tensor(CODES, dtype=torch.uint8)
    b = S.Float8Buffer(1, 4, data=codes, scales=torch.ones(1), device="cpu")
    assert b.ptr() == codes.data_ptr()


@pytest.mark.parametrize("data", [np.float32(VALUES), np.float64(VALUES), np.int8([1, -1, 4, 0]), np.int64(CODES), torch.tensor(VALUES), torch.tensor(VALUES).half(),
                                  torch.tensor(CODES), torch.tensor([1, -1, 4, 0], dtype=torch.int8), torch.tensor(VALUES).to(torch.float8_e5m2), VALUES, CODES],
                         ids=str)
def test_numbers_are_refused(data):
    with pytest.raises(ValueError, match="codes"):
        S.Float8Buffer(1, 4, data=data, scales=torch.ones(1), device="cpu")


@pytest.mark.parametrize("rows,columns,block_rows", [(1, 4, 1), (3, 272, 1), (130, 144, 128)])
def test_codes_without_scales(rows, columns, block_rows):
    b = S.Float8Buffer(rows, columns, block_rows, data=torch.full((rows, columns), 0x38, dtype=torch.uint8), device="cpu")
    assert (b.scales == 1).all() and (b.dequantized() == 1).all()
