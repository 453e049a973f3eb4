"""Block-scaled quantisation to e4m3: codes and scales are those of the definition, bit for bit."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu


def check(x, block_rows, stride=None, store=None):
    rows, columns = x.shape
    out = S.Float8Buffer(rows, columns, block_rows)
    S.QuantizeBlocks(rows, columns, U.buffer(x if store is None else store), out, input_stride=stride)
    torch.cuda.synchronize()
    codes, scales = U.quantize(x, block_rows)
    assert torch.equal(out.scales.view(scales.shape), scales)
    assert torch.equal(out.t.view(rows, columns).double(), codes)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,columns", [(1, 16), (1, 4096), (3, 128), (127, 144), (128, 112), (129, 272), (300, 2064), (1000, 128)])
def test_codes_and_scales(kind, block_rows, rows, columns):
    x = torch.randn(rows, columns, generator=U.generator(rows * columns), device="cuda")
    x[:, ::7] *= 40
    check(x.to(U.TYPES[kind]), block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_middles_between_codes(block_rows):
    """Whole multiples of small numbers: quotients that lie on, and right next to, the middle between two codes."""
    g = U.generator(1)
    x = torch.randint(-448, 449, (512, 256), generator=g, device="cuda").float()
    x[:, 0] = 448.0
    x[:, 128] = torch.where(torch.arange(512, device="cuda") % 2 == 0, 448.0, 447.0)
    check(x, block_rows)                              # scale 1: the quotient is the number
    check(x / 16, block_rows)
    check(x * 3.3e-7, block_rows)
    near = torch.nextafter(x, torch.full_like(x, torch.inf))
    check(near, block_rows)
    check(x.to(torch.bfloat16), block_rows)
    check((x * (7 / 448)).to(torch.float16), block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_zeros_and_the_smallest_and_largest_numbers(block_rows):
    g = U.generator(2)
    x = torch.randn(256, 384, generator=g, device="cuda")
    for scale in (0.0, 1e-45, 1e-40, 1e-38, 3e-36, 1e30, 1e38):
        v = (x * scale).clamp(-3.4e38, 3.4e38)
        check(v, block_rows)
    x[:, :128] = 0
    x[10, 130] = -0.0
    check(x, block_rows)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_values_that_are_not_finite(kind, block_rows):
    """They become NaN; the scale, and with it the other codes, are those of the block without them."""
    x = torch.randn(200, 272, generator=U.generator(3), device="cuda").to(U.TYPES[kind])
    bad = torch.zeros_like(x, dtype=torch.bool)
    for r, c, v in ((0, 0, torch.inf), (5, 130, -torch.inf), (5, 131, torch.nan), (140, 271, torch.nan), (199, 0, torch.inf)):
        x[r, c], bad[r, c] = v, True
    x[77, :128], bad[77, :128] = torch.nan, True      # a block with nothing else
    x[78, 128:256], bad[78, 128:256] = torch.inf, True
    out = S.Float8Buffer(200, 272, block_rows)
    S.QuantizeBlocks(200, 272, U.buffer(x), out)
    codes, scales = U.quantize(torch.where(bad, torch.zeros_like(x), x), block_rows)
    got = out.t.view(200, 272).double()
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], codes[~bad]) and torch.equal(out.scales.view(scales.shape), scales)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("stride,skip", [(160, 0), (160, 3), (147, 0), (145, 1)])
def test_rows_apart_and_any_alignment(kind, block_rows, stride, skip):
    rows, columns = 150, 144
    store = torch.randn(skip + rows * stride, generator=U.generator(4), device="cuda").to(U.TYPES[kind])[skip:]
    check(store.view(rows, stride)[:, :columns], block_rows, stride, store)


def test_what_lies_behind_is_left():
    x = torch.randn(130, 144, device="cuda")
    codes = torch.full((130 * 144 + 32,), 1, dtype=torch.uint8, device="cuda")
    scales = torch.full((4 + 5,), 7.0, device="cuda")
    _lib.check(_lib.lib().small_b200_quantize_blocks_f8(130, 144, 128, 0, x.data_ptr(), 0, codes.data_ptr(), scales.data_ptr(),
                                                        torch.cuda.current_stream().cuda_stream))
    assert (codes[130 * 144:] == 1).all() and (scales[4:] == 7).all() and (scales[:4] != 7).all()
