"""Dense layers on e4m3 operands whose rows end inside 16 bytes, begin anywhere, or end inside a tile, in the kernel for many rows, against 64 bits."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("K,apart,skip", [(4200, 4200, 0), (4204, 4208, 0), (4202, 4208, 0), (4201, 4201, 0), (4200, 4200, 1), (4200, 4203, 0), (4225, 4232, 0),
                                          (4104, 4104, 0)])
@pytest.mark.parametrize("partial", [False, True])
@pytest.mark.parametrize("rows", [290, 1000])
def test_rows_of_the_output(kind, K, apart, skip, partial, rows):
    C_ = 272
    x, w, g = U.operand(rows, C_, 1, 13), U.operand(K, C_, 128, 14), U.generator(15)
    b = torch.randn(K, generator=g, device="cuda") if partial else None
    store = torch.full((skip + rows * apart + 64,), torch.nan, device="cuda", dtype=U.TYPES[kind])
    y = store[skip:]
    got = torch.as_strided(y, (rows, K), (apart, 1))
    got.copy_(torch.randn(rows, K, generator=g, device="cuda") * 8)
    old = got.clone()
    mask = torch.ones_like(store, dtype=torch.bool)
    torch.as_strided(mask[skip:], (rows, K), (apart, 1)).zero_()
    S.Dense_Bias_Activation(K, C_, x, w, b, U.buffer(y), activation=2, negative_slope=0.5, partial=partial, batch=rows, output_stride=apart)
    assert _lib.device_status() == 0 and _lib.last_kernel().startswith("dense_f8_many_kernel")
    want, size = U.dense(x, w, b, 2, 0.5, old if partial else None)
    tolerance = U.dense_tolerance(want, size, C_, U.TYPES[kind])
    assert (((got.double() - want).abs() <= tolerance) | U.overflows(got, want, tolerance, U.TYPES[kind])).all()
    assert store[mask].isnan().all()
