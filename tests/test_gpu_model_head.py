"""The head of a model that answers: activations are quantised, two dense layers give the logits, and the answer is read from them."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,hidden,inner,classes", [(1, 512, 1024, 5003), (37, 256, 640, 1000), (200, 384, 512, 3001)])
def test_quantize_dense_logprobs(rows, hidden, inner, classes):
    g = U.generator(rows)
    top, padded = 7, classes + (-classes) % 8
    x = (torch.randn(rows, hidden, generator=g, device="cuda") * 2).to(torch.bfloat16)
    w1 = torch.randn(inner, hidden, generator=g, device="cuda") / hidden ** 0.5
    w2 = torch.randn(classes, inner, generator=g, device="cuda") / inner ** 0.5 * 4
    b1 = torch.randn(inner, generator=g, device="cuda") * 0.1
    tokens = torch.randint(classes, (rows,), generator=g, device="cuda")
    q1, q2 = S.Float8Buffer(inner, hidden, 128), S.Float8Buffer(classes, inner, 128)
    S.QuantizeBlocks(inner, hidden, S.FloatBuffer(data=w1), q1)
    S.QuantizeBlocks(classes, inner, S.FloatBuffer(data=w2), q2)
    qx, qh = S.Float8Buffer(rows, hidden), S.Float8Buffer(rows, inner)
    h, logits = S.BFloat16Buffer(rows * inner), S.FloatBuffer(rows * padded)
    lp, ent, tv, ti = S.FloatBuffer(rows), S.FloatBuffer(rows), S.FloatBuffer(rows * top), torch.empty(rows * top, dtype=torch.int32, device="cuda")
    bx, bias = S.BFloat16Buffer(data=x), S.FloatBuffer(data=b1)

    def answer():
        S.QuantizeBlocks(rows, hidden, bx, qx)
        S.Dense_Bias_Activation(inner, hidden, qx, q1, bias, h, activation=S.ACT_RELU, batch=rows)
        S.QuantizeBlocks(rows, inner, h, qh)
        S.Dense_Bias_Activation(classes, inner, qh, q2, None, logits, batch=rows, output_stride=padded)
        S.LogProbabilities(rows, classes, logits, tokens, lp, ent, tv, ti, top=top, row_stride=padded)

    answer()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    # each step against the plain form on what the step before it gave
    assert torch.equal(qx.t.view(rows, hidden).double(), U.quantize(x, 1)[0])
    want, size = U.dense(qx, q1, b1, S.ACT_RELU)
    assert ((h.t.view(rows, inner).double() - want).abs() <= U.dense_tolerance(want, size, hidden, torch.bfloat16)).all()
    assert torch.equal(qh.t.view(rows, inner).double(), U.quantize(h.t.view(rows, inner), 1)[0])
    want, size = U.dense(qh, q2)
    got = logits.t.view(rows, padded)[:, :classes]
    assert ((got.double() - want).abs() <= U.dense_tolerance(want, size, inner, torch.float32)).all()
    w_lp, w_h, w_tv, w_ti = U.logprobs(got, tokens, top)
    assert torch.equal(ti.view(rows, top).long(), w_ti)
    for a, b in ((lp.t, w_lp), (ent.t, w_h), (tv.t.view(rows, top), w_tv)):
        assert ((a.double() - b).abs() <= 1e-4 * (1 + b.abs())).all()
    # the whole run as one graph
    first = [t.clone() for t in (lp.t, ent.t, tv.t, ti)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        answer()
    for t in (lp.t, ent.t, tv.t, ti):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, (lp.t, ent.t, tv.t, ti)))
