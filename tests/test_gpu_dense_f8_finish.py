"""Bias, activation and old values of dense layers on e4m3 operands where a pair of CTAs has several tiles, against 64 bits."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu

ROWS, K, C_ = 2565, 4100, 272      # 11 x 17 tiles of 256 x 256: two and a half for each pair of CTAs, the last ones cut short both ways


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("apart", [0, 3, 28])
@pytest.mark.parametrize("act,partial,bias", [(1, False, True), (2, False, True), (2, False, False), (0, True, False), (2, True, True)])
def test_several_tiles(kind, apart, act, partial, bias):
    """The bias begins on any 4-byte boundary and rows lie any distance apart; old values behind the rows are NaN and stay."""
    x, w, g = U.operand(ROWS, C_, 1, 3), U.operand(K, C_, 128, 4), U.generator(5)
    b = torch.randn(K + 1, generator=g, device="cuda")[1:] * 4 if bias else None
    y = (torch.randn((ROWS + 1) * (K + apart), generator=g, device="cuda") * 8).to(U.TYPES[kind]).view(ROWS + 1, K + apart)
    y[:, K:] = torch.nan
    y[ROWS] = torch.nan
    old = y[:ROWS, :K].clone()
    flat = y.view(-1)
    S.Dense_Bias_Activation(K, C_, x, w, b, U.buffer(flat), activation=act, negative_slope=0.25, partial=partial, batch=ROWS, output_stride=K + apart)
    assert _lib.device_status() == 0 and _lib.last_kernel().startswith("dense_f8_many_kernel")
    want, size = U.dense(x, w, b, act, 0.25, old if partial else None)
    got = y[:ROWS, :K]
    tolerance = U.dense_tolerance(want, size, C_, U.TYPES[kind])
    assert (((got.double() - want).abs() <= tolerance) | U.overflows(got, want, tolerance, U.TYPES[kind])).all()
    assert y[ROWS].isnan().all() and y[:, K:].isnan().all()


@pytest.mark.parametrize("act", [0, 1, 2])
def test_infinities_of_the_bias_and_of_old_values(act):
    x, w = U.operand(ROWS, C_, 1, 3), U.operand(K, C_, 128, 4)
    b = torch.zeros(K, device="cuda")
    b[7], b[2049], b[K - 1] = torch.inf, -torch.inf, torch.nan
    y = torch.zeros(ROWS, K, device="cuda", dtype=torch.bfloat16)
    y[300, 5], y[2000, 6], y[ROWS - 1, 8] = torch.inf, -torch.inf, torch.nan
    S.Dense_Bias_Activation(K, C_, x, w, b, U.buffer(y), activation=act, negative_slope=0.5, partial=True, batch=ROWS)
    low = 0 if act == 1 else -torch.inf
    assert (y[:, 7] == torch.inf).all() and (y[:, 2049] == low).all() and y[:, K - 1].isnan().all()
    assert y[300, 5] == torch.inf and y[2000, 6] == low and y[ROWS - 1, 8].isnan()
    fine = torch.ones_like(y, dtype=torch.bool)
    fine[:, [7, 2049, K - 1]] = False
    fine[300, 5] = fine[2000, 6] = fine[ROWS - 1, 8] = False
    assert y[fine].isfinite().all()


def test_the_same_bits_every_time_and_beside_another_call():
    x, w, b = U.operand(ROWS, C_, 1, 3), U.operand(K, C_, 128, 4), S.FloatBuffer(data=torch.randn(K, device="cuda"))
    def call(y, stream=None):
        S.Dense_Bias_Activation(K, C_, x, w, b, U.buffer(y), activation=1, partial=True, batch=ROWS, stream=stream)
    start = torch.randn(ROWS, K, generator=U.generator(1), device="cuda").bfloat16()
    want, ys, streams = start.clone(), [start.clone() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        call(want)
    torch.cuda.synchronize()
    for _ in range(3):
        for y, s in zip(ys, streams):
            call(y, s)
    torch.cuda.synchronize()
    assert torch.equal(ys[0], want) and torch.equal(ys[1], want) and _lib.device_status() == 0
