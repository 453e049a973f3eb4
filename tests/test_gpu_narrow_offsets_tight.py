"""Log-probabilities where offsets pass 32 bits, within the tolerance of what reads a row: a CTA (256 threads) or, for many rows of few classes, a warp (32 lanes)."""
import pytest
import torch

from smallframework_b200 import interface as S
from tests import narrow_util as U
from tests.test_gpu_logprobs import compare
from tests.test_gpu_logprobs import tolerance as of_cta
from tests.test_gpu_logprobs_many_rows import tolerance as of_warp

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,classes,stride,warp", [(17000, 131072, 131072, False), (9, 5000, 2 ** 28 + 3, False), (700, 1000, 2 ** 22 + 1, True)])
def test_logits(rows, classes, stride, warp):
    assert (rows - 1) * stride + classes > 2 ** 31
    x = torch.zeros((rows - 1) * stride + classes, device="cuda", dtype=torch.bfloat16)
    view = torch.as_strided(x, (rows, classes), (stride, 1))
    at = torch.tensor([0, rows // 2, rows - 2, rows - 1], device="cuda")
    view[at] = torch.randn(4, classes, device="cuda", generator=U.generator(1)).bfloat16() * 3
    tokens = torch.randint(classes, (rows,), generator=U.generator(2), device="cuda")
    lp, h = S.FloatBuffer(rows), S.FloatBuffer(rows)
    tv, ti = S.FloatBuffer(rows * 8), torch.empty(rows * 8, dtype=torch.int32, device="cuda")
    S.LogProbabilities(rows, classes, U.buffer(x), tokens, lp, h, tv, ti, top=8, row_stride=stride)
    w_lp, w_h, w_tv, w_ti = U.logprobs(view[at].float(), tokens[at], 8)
    tol = (lambda want: of_warp(want, classes)) if warp else (lambda want: of_cta(x, want, classes))
    assert torch.equal(ti.view(rows, 8)[at].long(), w_ti)
    compare(lp.t[at], w_lp, tol(w_lp)[0])
    compare(tv.t.view(rows, 8)[at], w_tv, tol(w_tv)[0])
    compare(h.t[at], w_h, torch.full_like(w_h, tol(w_lp)[1]))
    # one row's logits in another's place would be far outside
    assert (w_lp - w_lp.roll(1)).abs().min() > 10 * tol(w_lp)[0].max()
