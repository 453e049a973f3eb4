"""The layers of narrow types at the ends of their sizes: what a 32-bit count of tiles or blocks would not hold is refused before any CUDA call."""
import ctypes as C

import pytest

from smallframework_b200 import _lib

P = 1 << 20  # an address that is never followed


@pytest.mark.parametrize("rows,K,C_", [(1, 2 ** 31 - 1, 16), (2 ** 31 - 1, 1, 16), (1, 1, 2 ** 31 - 16), (1, 2 ** 31 - 512, 16), (2 ** 31 - 512, 1, 16)])
def test_dense(rows, K, C_):
    D = _lib.DenseLayer(rows=rows, K=K, C=C_, out_type=_lib.TYPE_F32)
    assert _lib.lib().small_b200_dense_f8(C.byref(D), P, P, P, P, None, P, None) == _lib.INVALID_ARGUMENT
    assert "too many tiles" in _lib.lib().small_b200_last_error().decode()


@pytest.mark.parametrize("rows,columns,block_rows", [(128, 2 ** 31 - 16, 1), (2 ** 31 - 1, 2 ** 31 - 16, 128), (2 ** 31 - 1, 2 ** 31 - 112, 1)])
def test_quantize(rows, columns, block_rows):
    assert _lib.lib().small_b200_quantize_blocks_f8(rows, columns, block_rows, _lib.TYPE_BF16, P, 0, P, P, None) == _lib.INVALID_ARGUMENT
    assert "too many blocks" in _lib.lib().small_b200_last_error().decode()
