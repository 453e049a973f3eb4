"""Calls that read at once what the call before them wrote, where rows begin on no 32-byte boundary and a layer adds to its old output: two CTAs then read and write
the two ends of one sector, and the next kernel, which may exist by then, reads both."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu

STEPS = 12


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,K,C_", [(1, 1001, 512), (5, 333, 256), (24, 2067, 1040), (40, 515, 4096), (70, 1003, 272), (300, 4109, 272), (1100, 2501, 272),
                                       (3, 2 * 148 * 128 + 645, 2048)])
def test_old_outputs_read_by_the_next_call(kind, rows, K, C_):
    """x -> e4m3 -> y += W x -> log-probabilities of y, and y's first columns as e4m3 -> the next x.  With and without waits between the calls, and as a graph."""
    g, cut = U.generator(K), K // 16 * 16
    w, back = S.Float8Buffer(K, C_, 128), S.Float8Buffer(C_, cut, 128)
    S.QuantizeBlocks(K, C_, U.buffer(torch.randn(K, C_, generator=g, device="cuda") / C_ ** 0.5), w)
    S.QuantizeBlocks(C_, cut, U.buffer(torch.randn(C_, cut, generator=g, device="cuda") * (0.05 / cut ** 0.5)), back)
    first = torch.randn(rows, C_, generator=g, device="cuda")
    tokens = torch.randint(K, (rows,), generator=g, device="cuda")
    x, q, p = first.clone(), S.Float8Buffer(rows, C_), S.Float8Buffer(rows, cut)
    y = torch.zeros(rows * K, device="cuda", dtype=U.TYPES[kind])
    lp, h, tv, ti = (torch.zeros(STEPS, rows, device="cuda"), torch.zeros(STEPS, rows, device="cuda"), torch.zeros(STEPS, rows * 4, device="cuda"),
                     torch.zeros(STEPS, rows * 4, dtype=torch.int32, device="cuda"))

    def run(wait):
        x.copy_(first)
        y.zero_()
        for n in range(STEPS):
            S.QuantizeBlocks(rows, C_, U.buffer(x), q)
            wait()
            S.Dense_Bias_Activation(K, C_, q, w, None, U.buffer(y), partial=True, batch=rows)
            wait()
            S.LogProbabilities(rows, K, U.buffer(y), tokens, U.buffer(lp[n]), U.buffer(h[n]), U.buffer(tv[n]), ti[n], top=4)
            wait()
            S.Dense_Bias_Activation(K, C_, q, w, None, U.buffer(y), partial=True, batch=rows)
            wait()
            S.QuantizeBlocks(rows, cut, U.buffer(y), p, input_stride=K)
            wait()
            S.Dense(C_, cut, p, back, U.buffer(x), batch=rows)
            wait()

    outs = (x, y, lp, h, tv, ti)
    run(torch.cuda.synchronize)
    want = [t.clone() for t in outs]
    assert all(t.isfinite().all() for t in want[:4]) and not torch.equal(want[2][0], want[2][-1])
    for _ in range(3):
        run(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(lambda: None)
    for _ in range(3):
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("rows", [8, 600, 3000, 3552, 3553, 9000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_of_a_warp_each_behind_what_writes_them(rows, kind):
    """Log-probabilities that start early (grids that are resident at once) and that do not, behind a dense layer and before one that writes the logits anew."""
    K, C_ = 701, 128
    w, xs = U.operand(K, C_, 128, 1, spread_of_scales=0.0), [U.operand(rows, C_, 1, s, spread_of_scales=0.0) for s in (2, 3, 4)]
    y, tokens = torch.zeros(rows * K, device="cuda", dtype=U.TYPES[kind]), torch.arange(rows, device="cuda") % K
    out = [(torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(rows * 3, device="cuda"), torch.zeros(rows * 3, dtype=torch.int32, device="cuda"))
           for _ in range(6)]

    def run(wait):
        for n, (lp, h, tv, ti) in enumerate(out):
            S.Dense(K, C_, xs[n % 3], w, U.buffer(y), batch=rows)
            wait()
            S.LogProbabilities(rows, K, U.buffer(y), tokens, U.buffer(lp), U.buffer(h), U.buffer(tv), ti, top=3)
            wait()

    run(torch.cuda.synchronize)
    want = [[t.clone() for t in o] for o in out]
    assert not torch.equal(want[0][0], want[1][0])
    for _ in range(5):
        for o in out:
            for t in o:
                t.zero_()
        run(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, v in zip(out, want) for a, b in zip(o, v))
    assert _lib.device_status() == 0
