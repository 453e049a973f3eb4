"""Log-probabilities of so many rows that each goes to a warp, however long it is, and of one row fewer, which go to a CTA each."""
import pytest
import torch

from tests import narrow_util as U
from tests.test_gpu_logprobs import logits
from smallframework_b200 import interface as S

pytestmark = pytest.mark.gpu


def tolerance(x_lp, classes):
    """Absolute: an exponential is off by 2^-22 of itself and by 2^-23 |t| (its argument's two roundings; a row's mean |t| is at most 2 ln(classes) + 2);
    a lane adds at most ceil(classes / 32) + 16 of them, one rounding each, and 16 merges follow.  T has the same and a rounding more a term."""
    depth = 2.0 * torch.log(torch.tensor(float(classes))).item() + 2
    delta = 2.0 ** -22 + (depth + 2) * 2.0 ** -23 + (classes / 32 + 40) * 2.0 ** -24
    return delta + 2.0 ** -22 * (x_lp.abs().clamp(max=1e30) + 1), delta * (1 + 3 * depth)


def check(x, top, tokens):
    rows, classes = x.shape
    lp, h = S.FloatBuffer(rows), S.FloatBuffer(rows)
    tv, ti = S.FloatBuffer(rows * top), torch.full((rows * top,), -7, dtype=torch.int32, device="cuda")
    S.LogProbabilities(rows, classes, U.buffer(x), tokens, lp, h, tv, ti, top=top)
    torch.cuda.synchronize()
    w_lp, w_h, w_tv, w_ti = U.logprobs(x, tokens, top)
    for got, want, tol in ((lp.t, w_lp, tolerance(w_lp, classes)[0]), (h.t, w_h, torch.full_like(w_h, tolerance(w_lp, classes)[1])),
                           (tv.t.view(rows, top), w_tv, tolerance(w_tv, classes)[0])):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        assert ((got.double() - want).abs() <= tol)[want.isfinite()].all()
    assert torch.equal(ti.view(rows, top).long(), w_ti)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes,top", [(768, 8), (769, 32), (1500, 0), (4001, 5), (8192, 32), (8193, 3), (16384, 8), (16385, 2)])
@pytest.mark.parametrize("more", [0, 1])
def test_sizes(kind, classes, top, more):
    rows = 4 * torch.cuda.get_device_properties(0).multi_processor_count + more
    check(logits(rows, classes, kind, seed=classes), top, torch.randint(classes, (rows,), generator=U.generator(rows), device="cuda"))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [2500, 8191])
def test_rows_that_are_hard(kind, classes):
    """Equal, ascending, descending, masked, empty and broken rows, among ordinary ones and in the last rows of a CTA that has fewer."""
    rows = 4 * torch.cuda.get_device_properties(0).multi_processor_count + 11
    x = logits(rows, classes, kind, seed=2)
    low = torch.finfo(x.dtype).min
    for at in (0, 100, rows - 12):
        x[at] = 1.5
        x[at + 1] = torch.linspace(-20, 20, classes, device="cuda")
        x[at + 2] = x[at + 1].flip(0)
        x[at + 3, torch.rand(classes, device="cuda", generator=U.generator(1)) < 0.95] = low
        x[at + 4, torch.rand(classes, device="cuda", generator=U.generator(2)) < 0.95] = -torch.inf
        x[at + 5] = -torch.inf
        x[at + 6] = low
        x[at + 7], x[at + 7, classes - 2] = -torch.inf, 2.0
        x[at + 8, classes // 3] = torch.nan
        x[at + 9, classes - 1] = torch.inf
        x[at + 10] = -5.0
        x[at + 10, torch.arange(0, classes, device="cuda") // 8 % 32 == 3] = 5.0
    check(x, 16, torch.full((rows,), classes - 2, device="cuda"))
