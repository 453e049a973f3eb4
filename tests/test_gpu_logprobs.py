"""Log-probabilities of given classes, entropy and the best alternatives, against 64 bits."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu


def tolerance(x, want_lp, classes):
    """Absolute, for log S: an exponential is off by 2^-22 of itself (the unit) and by 2^-23 |t| (its argument's two roundings), which a
    row's mean |t| <= 2 ln(classes) + 2 bounds for the sum; a thread adds at most ceil(classes / 256) + 16 of them, one rounding each, and 16 merges
    follow.  T has the same and a rounding more a term."""
    depth = 2.0 * torch.log(torch.tensor(float(classes))).item() + 2
    delta = 2.0 ** -22 + (depth + 2) * 2.0 ** -23 + (classes / 256 + 40) * 2.0 ** -24
    lp = delta + 2.0 ** -22 * (want_lp.abs().clamp(max=1e30) + 1)
    return lp, delta * (1 + 3 * depth)


def compare(got, want, tol):
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    assert ((got.double() - want).abs() <= tol)[fine].all(), (got.double() - want).abs()[fine].max().item()


def run(x, top=5, tokens=None, stride=None, store=None, kinds=torch.int64):
    rows, classes = x.shape
    if tokens is None:
        tokens = torch.randint(classes, (rows,), generator=U.generator(rows), device="cuda")
    lp, h = S.FloatBuffer(rows), S.FloatBuffer(rows)
    tv, ti = S.FloatBuffer(rows * top), torch.full((rows * top,), -7, dtype=torch.int32, device="cuda")
    S.LogProbabilities(rows, classes, U.buffer(x if store is None else store), tokens.to(kinds), lp, h, tv, ti, top=top, row_stride=stride)
    torch.cuda.synchronize()
    w_lp, w_h, w_tv, w_ti = U.logprobs(x, tokens.long(), top)
    t_lp, t_h = tolerance(x, w_lp, classes)
    compare(lp.t, w_lp, t_lp)
    compare(h.t, w_h, torch.full_like(w_h, t_h))
    assert torch.equal(ti.view(rows, top).long(), w_ti)
    compare(tv.t.view(rows, top), w_tv, tolerance(x, w_tv, classes)[0])
    return lp.t, h.t, tv.t, ti


def logits(rows, classes, kind, seed=0, size=3.0):
    return (torch.randn(rows, classes, generator=U.generator(seed), device="cuda") * size).to(U.TYPES[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,classes,top", [(1, 1, 1), (3, 2, 2), (2, 7, 7), (1, 8, 8), (5, 31, 31), (4, 33, 32), (1, 64, 32), (7, 255, 1), (3, 1000, 5), (2, 1001, 0), (2, 4099, 20),
                                              (9, 16384, 32), (300, 2050, 8), (2, 50257, 10), (1, 131072, 20), (600, 300, 3)])
def test_sizes(kind, rows, classes, top):
    run(logits(rows, classes, kind, seed=classes), top)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [40, 1000, 70000])
def test_equal_logits_go_to_the_lowest_class(kind, classes):
    x = logits(4, classes, kind, seed=3)
    x[0] = 1.5                                           # all alike
    x[1] = (x[1].float() / 2).round().to(x.dtype)        # a few values
    x[2, ::2], x[2, 1::2] = 0.0, -0.0                    # zeros of both signs are alike
    x[3] = -torch.inf
    x[3, classes // 2:classes // 2 + 3] = 2.0            # fewer than asked for are allowed
    run(x, 32)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [100, 5000, 200000])
def test_orders_that_fill_the_candidates(kind, classes):
    """Ascending and descending rows, and one whose largest logits all belong to one thread or to a few."""
    x = torch.empty(4, classes, device="cuda")
    x[0] = torch.linspace(-20, 20, classes, device="cuda")
    x[1] = x[0].flip(0)
    x[2] = -5.0
    at = torch.arange(0, classes, device="cuda") // 8 % 256 == 3
    x[2, at] = torch.randn(int(at.sum()), generator=U.generator(5), device="cuda") + 5
    x[3] = torch.arange(classes, device="cuda") // 4 % 256 // 16 * 1.0
    run(x.to(U.TYPES[kind]), 32)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [50, 3000, 140000])
def test_masks(kind, classes):
    low = torch.finfo(U.TYPES[kind]).min
    x = logits(8, classes, kind, seed=8)
    x[0, 1:] = -torch.inf                                # one class
    x[1, : classes - 1] = -torch.inf
    x[2, torch.rand(classes, device="cuda", generator=U.generator(1)) < 0.9] = low
    x[3, torch.rand(classes, device="cuda", generator=U.generator(2)) < 0.9] = -torch.inf
    x[4] = -torch.inf                                    # nothing
    x[5] = low                                           # masked by the lowest value: all alike
    x[6, : classes // 2], x[6, classes // 2:] = -torch.inf, low
    tokens = torch.tensor([0, 0, classes - 1, 5, 3, 1, 0, -1], device="cuda")
    lp, h, tv, ti = run(x, 16, tokens)
    assert lp[0] == 0 and h[0] == 0 and lp[1] == -torch.inf and lp[4] == -torch.inf and h[4] == 0 and lp[7] == 0


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes", [37, 2500, 131072])
def test_nan_and_infinities(kind, classes):
    """A row with NaN or plus infinity has no distribution, wherever it stands; its neighbours are as they were."""
    x = logits(7, classes, kind, seed=4)
    x[1, 0] = torch.nan
    x[2, classes - 1] = torch.nan
    x[3, classes // 2] = torch.inf
    x[4] = torch.nan
    x[5], x[5, 3] = -torch.inf, torch.nan
    lp, h, tv, ti = run(x, 8)
    assert lp[1:6].isnan().all() and h[1:6].isnan().all() and lp[[0, 6]].isfinite().all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_large_and_confident_logits(kind):
    x = logits(6, 5000, kind, seed=6)
    x[0] += 3e4
    x[1] *= 1e4
    x[2, 17] = 1e30 if kind == "bf16" else 3e38
    x[3] -= 3e4
    x[4, 9] = 60.0
    x[5, 9] = 25.0
    lp, h, _, _ = run(x, 4, torch.full((6,), 9, device="cuda"))
    assert (h >= 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("classes,stride,skip", [(1000, 1024, 0), (1001, 1003, 1), (5000, 5001, 5), (40001, 40001, 3), (3, 3, 1)])
def test_rows_apart_and_any_alignment(kind, classes, stride, skip):
    """What lies between the rows is not a class."""
    rows = 5
    store = torch.full((skip + rows * stride + 8,), 99.0, device="cuda", dtype=U.TYPES[kind])[skip:]
    x = store[:rows * stride].view(rows, stride)[:, :classes]
    x.copy_(logits(rows, classes, kind, seed=10))
    run(x, 3, stride=stride, store=store)


def test_tokens_of_both_sizes_and_outside():
    x = logits(5, 900, "f32")
    for kinds in (torch.int32, torch.int64):
        lp, _, _, _ = run(x, 2, torch.tensor([0, 899, 900, -1, -100], device="cuda"), kinds=kinds)
        assert lp[2].isnan() and (lp[3:] == 0).all()
    lp, _, _, _ = run(x, 2, torch.tensor([1 << 40, -(1 << 40), 0, 1, 2], device="cuda"))
    assert lp[0].isnan() and lp[1] == 0


@pytest.mark.parametrize("classes", [500, 60000])
def test_each_output_alone(classes):
    x = logits(4, classes, "bf16")
    tokens = torch.tensor([1, 2, 3, 4], device="cuda")
    lp, h, tv, ti = run(x, 6, tokens)
    buf, rows = U.buffer(x), 4
    a, b, c = S.FloatBuffer(rows), S.FloatBuffer(rows), S.FloatBuffer(rows * 6)
    d = torch.empty(rows * 6, dtype=torch.int32, device="cuda")
    S.LogProbabilities(rows, classes, buf, tokens, a)
    S.LogProbabilities(rows, classes, buf, None, None, b)
    S.LogProbabilities(rows, classes, buf, None, None, None, c, top=6)
    S.LogProbabilities(rows, classes, buf, None, None, None, None, d, top=6)
    assert torch.equal(a.t, lp) and torch.equal(b.t, h) and torch.equal(c.t, tv) and torch.equal(d, ti)


@pytest.mark.parametrize("rows,classes", [(1, 131072), (40, 9000)])
def test_two_streams_and_a_replayed_graph(rows, classes):
    x, other = logits(rows, classes, "f16", 1), logits(rows, classes, "f16", 2)
    tokens = torch.arange(rows, device="cuda")
    want = [run(v, 9, tokens) for v in (x, other)]
    outs = [(S.FloatBuffer(rows), S.FloatBuffer(rows), S.FloatBuffer(rows * 9), torch.empty(rows * 9, dtype=torch.int32, device="cuda")) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, v, o in zip(streams, (x, other), outs):
            S.LogProbabilities(rows, classes, U.buffer(v), tokens, *o, top=9, stream=s)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(p.t if isinstance(p, S.FloatBuffer) else p, q) for p, q in zip(o, w))
    graph, buf = torch.cuda.CUDAGraph(), U.buffer(x)
    with torch.cuda.graph(graph):
        S.LogProbabilities(rows, classes, buf, tokens, *outs[0], top=9)
    x.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p.t if isinstance(p, S.FloatBuffer) else p, q) for p, q in zip(outs[0], want[1]))
