"""The best alternatives where many logits are equal, for every number of CTAs to a row: the classes have to be the lowest ones."""
import pytest
import torch

from smallframework_b200 import interface as S
from tests import narrow_util as U
from tests.test_gpu_logprobs import tolerance

pytestmark = pytest.mark.gpu


def alternatives(x, top, stream=None):
    rows, classes = x.shape
    tv, ti = torch.empty(rows * top, device="cuda"), torch.full((rows * top,), -7, dtype=torch.int32, device="cuda")
    S.LogProbabilities(rows, classes, U.buffer(x), None, None, None, tv, ti, top=top, stream=stream)
    return tv.view(rows, top), ti.view(rows, top)


def tied(rows, classes, kind):
    """Kinds of rows in turn: all alike, two values, a few values, two values of which the larger is rare, runs of equal values, masked but for a few,
    masked whole by either way, and the largest values all in steps of one thread."""
    x = torch.zeros(rows, classes, device="cuda")
    i = torch.arange(classes, device="cuda")
    u = torch.rand(rows, classes, generator=U.generator(rows + classes), device="cuda")
    low = torch.finfo(U.TYPES[kind]).min
    for r in range(rows):
        k = r % 9
        if k == 1:
            x[r] = (u[r] < 0.5).float()
        elif k == 2:
            x[r] = (u[r] * 5).floor()
        elif k == 3:
            x[r] = (u[r] < 0.004).float()
        elif k == 4:
            x[r] = (i // 7 % 13).float()
        elif k == 5:
            x[r] = torch.where(u[r] < 3.0 / classes, 1.0, -torch.inf)
        elif k == 6:
            x[r] = -torch.inf
        elif k == 7:
            x[r] = low
        elif k == 8:
            x[r] = (i // 8 % 256 == r % 256).float()
    return x.to(U.TYPES[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,classes", [(9, 5000), (9, 50257), (9, 140000), (60, 33000), (70, 132001), (160, 131072), (310, 20001)])
@pytest.mark.parametrize("top", [1, 9, 32])
def test_the_lowest_classes(kind, rows, classes, top):
    x = tied(rows, classes, kind)
    tv, ti = alternatives(x, top)
    want_v, want = U.logprobs(x, torch.zeros(rows, dtype=torch.long, device="cuda"), top)[2:]
    assert torch.equal(ti.long(), want)
    assert torch.equal(tv.isinf(), want_v.isinf()) and not tv.isnan().any()
    fine = want_v.isfinite()
    assert ((tv.double() - want_v).abs() <= tolerance(x, want_v, classes)[0])[fine].all()


def test_two_streams_at_once():
    x = [tied(9, 60000, "bf16"), tied(160, 140000, "f16")]
    want = [alternatives(v, 20) for v in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = [alternatives(v, 20, stream=s) for v, s in zip(x, streams)]
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
