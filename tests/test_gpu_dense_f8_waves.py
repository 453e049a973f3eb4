"""Dense layers on e4m3 operands with more tiles than the device holds at once, a few rows: two launches side by side, and what comes before and behind them."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu

K = 2 * 148 * 128 + 5 * 128 + 40


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 24, 60])
@pytest.mark.parametrize("C_", [2048, 4112])
@pytest.mark.parametrize("outputs,partial", [(K, False), (K, True), (2 * K + 9, False), (2 * 148 * 128, False)])
def test_outputs(kind, rows, C_, outputs, partial):
    x, w, g = U.operand(rows, C_, 1, 3), U.operand(outputs, C_, 128, 4), U.generator(5)
    b = torch.randn(outputs, generator=g, device="cuda")
    y = (torch.randn(rows, outputs, generator=g, device="cuda") * 8).to(U.TYPES[kind])
    old = y.clone()
    S.Dense_Bias_Activation(outputs, C_, x, w, b, U.buffer(y), activation=2, negative_slope=0.25, partial=partial, batch=rows)
    assert _lib.device_status() == 0
    want, size = U.dense(x, w, b, 2, 0.25, old if partial else None)
    assert ((y.double() - want).abs() <= U.dense_tolerance(want, size, C_, U.TYPES[kind])).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_a_chain_of_calls(rows):
    """Every call reads what the one before it wrote, many times over, eagerly and as a graph: none may start on what is not there yet."""
    C_ = 2048
    wide, back = U.operand(K, C_, 128, 7, spread_of_scales=0.5), U.operand(C_, K // 16 * 16, 128, 8, spread_of_scales=0.5)
    x, a = torch.randn(rows, C_, generator=U.generator(9), device="cuda"), S.Float8Buffer(rows, C_)
    y, b, z = torch.zeros(rows, K, device="cuda", dtype=torch.bfloat16), S.Float8Buffer(rows, K // 16 * 16), torch.zeros(rows, C_, device="cuda")

    def step(wait):
        S.QuantizeBlocks(rows, C_, U.buffer(x), a)
        wait()
        S.Dense(K, C_, a, wide, U.buffer(y), batch=rows)
        wait()
        S.QuantizeBlocks(rows, K // 16 * 16, U.buffer(y), b, input_stride=K)
        wait()
        S.Dense(C_, K // 16 * 16, b, back, U.buffer(z), batch=rows)
        wait()
        x.copy_(z / z.abs().amax().clamp_min(1e-30))

    start = x.clone()
    for _ in range(5):
        step(torch.cuda.synchronize)
    want = x.clone()
    assert want.isfinite().all()
    x.copy_(start)
    for _ in range(5):
        step(lambda: None)
    torch.cuda.synchronize()
    assert torch.equal(x, want)
    x.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(lambda: None)
    x.copy_(start)
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, want) and _lib.device_status() == 0


def test_two_streams_at_once():
    C_, rows = 2048, 8
    w, xs = U.operand(K, C_, 128, 4), [U.operand(rows, C_, 1, s) for s in (1, 2)]
    want = [torch.empty(rows, K, device="cuda") for _ in xs]
    for x, y in zip(xs, want):
        S.Dense(K, C_, x, w, U.buffer(y), batch=rows)
    torch.cuda.synchronize()
    ys, streams = [torch.zeros(rows, K, device="cuda") for _ in xs], [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for x, y, s in zip(xs, ys, streams):
            S.Dense(K, C_, x, w, U.buffer(y), batch=rows, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(ys[0], want[0]) and torch.equal(ys[1], want[1]) and _lib.device_status() == 0
