"""Bias and old values of dense layers on e4m3 operands, as large as the products' sums: dropped, added twice, or taken from the next column or row they would be
far outside the tolerance in every column, which each test shows for itself."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu

WAVE = 2 * 148 * 128
# rows, outputs, inputs, elements between the ends of rows, the kernel
SIZES = [(1, 512, 4096, 0, "few"), (1, 4097, 1040, 3, "few"), (3, 130, 8192, 0, "few"), (16, 257, 272, 0, "few"), (24, 2049, 4112, 7, "few"), (40, 300, 2064, 0, "few"),
         (64, 1001, 2064, 0, "few"), (140, 640, 4096, 0, "few"), (333, 1001, 2064, 0, "few"),
         (1, WAVE + 685, 2048, 0, "few"), (24, WAVE + 685, 4112, 0, "few"), (60, 2 * WAVE + 9, 2048, 1, "few"),
         (1100, 2500, 272, 0, "many_kernel<256>"), (300, 4100, 1040, 4, "many_kernel<128>"), (2300, 2310, 400, 0, "many_kernel<128>"),
         (2565, 4100, 272, 3, "many"), (290, 4201, 272, 0, "many"), (1000, 4225, 272, 7, "many")]
EPILOGUES = [(0, False, True), (2, False, True), (1, False, True), (0, True, False), (2, True, True)]


def seen(want, without, tolerance, act):
    """Most of what is left out would show: in every column and in every row where the activation cuts nothing off, and in most of all places behind ReLU."""
    far = (want - without).abs() > 4 * tolerance
    if act != 1:
        return far.double().mean(0).min() > 0.9 and far.double().mean(1).min() > 0.9
    return far.double().mean() > 0.4 and (want.shape[0] < 64 or far.any(0).all())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act,partial,bias", EPILOGUES)
@pytest.mark.parametrize("rows,K,C_,apart,name", SIZES)
def test_bias_and_old_values(kind, act, partial, bias, rows, K, C_, apart, name):
    x, w, g = U.operand(rows, C_, 1, 3, spread_of_scales=0.0), U.operand(K, C_, 128, 4, spread_of_scales=0.0), U.generator(5)
    plain = U.dense(x, w)[0]
    rms = plain.square().mean().sqrt().item()
    signs = torch.where(torch.arange(K, device="cuda") % 2 == 0, 1.0, -1.0)  # neighbours differ by twice the sums' size at least
    b = signs * (1 + 2 * torch.rand(K, generator=g, device="cuda")) * rms if bias else None
    width = K + apart
    store = torch.full((rows * width + 64,), torch.nan, device="cuda", dtype=U.TYPES[kind])
    got = torch.as_strided(store, (rows, K), (width, 1))
    old = signs * torch.where(torch.arange(rows, device="cuda") % 2 == 0, 1.0, -1.0)[:, None] * (1 + 2 * torch.rand(rows, K, generator=g, device="cuda")) * rms
    got.copy_(old)
    old = got.clone() if partial else None
    S.Dense_Bias_Activation(K, C_, x, w, b, U.buffer(store), activation=act, negative_slope=0.25, partial=partial, batch=rows, output_stride=width)
    assert _lib.device_status() == 0 and _lib.last_kernel().startswith("dense_f8_" + name)
    want, size = U.dense(x, w, b, act, 0.25, old)
    tolerance = U.dense_tolerance(want, size, C_, U.TYPES[kind])
    if bias:
        assert seen(want, U.dense(x, w, None, act, 0.25, old)[0], tolerance, act)
    if partial:
        assert seen(want, U.dense(x, w, b, act, 0.25)[0], tolerance, act)
    assert ((got.double() - want).abs() <= tolerance).all()
    behind = torch.ones_like(store, dtype=torch.bool)
    torch.as_strided(behind, (rows, K), (width, 1)).zero_()
    assert store[behind].isnan().all()
