"""Square blocks with infinities and NaN among values of every kind, in 16 bits as in 32: as if those elements were zeros, but for their codes."""
import pytest
import torch

from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,columns,stride", [(300, 528, 528), (257, 144, 160), (1100, 2064, 2065)])
def test_values_that_are_not_finite(kind, block_rows, rows, columns, stride):
    x = torch.randn(rows, columns, generator=U.generator(rows), device="cuda").mul(torch.rand(rows, 1, generator=U.generator(1), device="cuda").mul(8).exp()).to(U.TYPES[kind])
    bad = torch.rand(rows, columns, generator=U.generator(2), device="cuda") < torch.tensor([0.0, 1e-4, 0.01], device="cuda")[torch.arange(rows, device="cuda") // 128 % 3][:, None]
    bad[-1] = True                                      # a row, and with rows = 257 a block, of nothing else
    what = torch.tensor([torch.inf, -torch.inf, torch.nan], device="cuda").to(x.dtype)[torch.randint(3, (rows, columns), generator=U.generator(3), device="cuda")]
    store = torch.full((rows * stride,), 7.0, device="cuda", dtype=x.dtype)
    torch.as_strided(store, (rows, columns), (stride, 1)).copy_(torch.where(bad, what, x))
    q = S.Float8Buffer(rows, columns, block_rows)
    S.QuantizeBlocks(rows, columns, U.buffer(store), q, input_stride=stride)
    want, scales = U.quantize(torch.where(bad, torch.zeros_like(x), x), block_rows)
    got = q.t.view(rows, columns).double()
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad]) and torch.equal(q.scales, scales.view(-1))
