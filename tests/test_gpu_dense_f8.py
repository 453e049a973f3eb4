"""Dense layers on e4m3 operands with block scales, against the same sums in 64 bits."""
import ctypes as C

import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu


def run(rows, K, C_, kind, seed=0, bias=True, act=0, slope=0.25, partial=False, stride=None):
    x, w = U.operand(rows, C_, 1, seed), U.operand(K, C_, 128, seed + 1)
    g = U.generator(seed + 2)
    b = torch.randn(K, generator=g, device="cuda") if bias else None
    apart = stride or K
    y = (torch.randn(rows * apart + 64, generator=g, device="cuda") * 8).to(U.TYPES[kind])
    before = y.clone()
    old = y[:rows * apart].view(rows, apart)[:, :K].clone()
    S.Dense_Bias_Activation(K, C_, x, w, None if b is None else S.FloatBuffer(data=b), U.buffer(y), activation=act, negative_slope=slope,
                            partial=partial, batch=rows, output_stride=stride)
    assert _lib.device_status() == 0
    got = y[:rows * apart].view(rows, apart)
    want, size = U.dense(x, w, b, act, slope, old if partial else None)
    off = (got[:, :K].double() - want).abs()
    tolerance = U.dense_tolerance(want, size, C_, U.TYPES[kind])
    assert ((off <= tolerance) | U.overflows(got[:, :K], want, tolerance, U.TYPES[kind])).all(), (off / tolerance).max().item()
    assert torch.equal(got[:, K:], before[:rows * apart].view(rows, apart)[:, K:]) and torch.equal(y[rows * apart:], before[rows * apart:])
    return off, size


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("K,C_", [(128, 128), (100, 144), (257, 16), (1, 256), (640, 1040)])
def test_rows_outputs_and_blocks_cut_short(rows, K, C_):
    run(rows, K, C_, "f32", seed=rows + K)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,K,C_", [(1, 512, 4096), (3, 130, 8192), (40, 300, 2064), (200, 513, 2048), (1000, 1001, 528)])
@pytest.mark.parametrize("act,partial,bias", [(0, False, False), (1, False, True), (2, True, True), (0, True, False)])
def test_types_activations_and_partial(kind, rows, K, C_, act, partial, bias):
    run(rows, K, C_, kind, seed=5, bias=bias, act=act, partial=partial)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,K,stride", [(5, 100, 101), (5, 100, 128), (150, 257, 264), (150, 257, 259), (130, 8, 8)])
def test_rows_of_the_output_apart(kind, rows, K, stride):
    run(rows, K, 384, kind, seed=9, stride=stride, partial=True, act=2)


@pytest.mark.parametrize("rows", [1, 60, 129, 700])
def test_many_tiles(rows):
    """More tiles than SMs, more blocks than stages."""
    run(rows, 148 * 256 + 40, 1280, "bf16", seed=3)


# Sizes that take the kernel for many rows: whole tiles, halves of tiles (the last of which begins behind the last output), and one after the other.
MANY = [(1100, 2500, 272, "<256>"), (300, 4100, 1040, "<128>"), (2300, 2310, 400, "<128>")]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act,partial,bias,apart", [(0, False, False, 0), (1, False, True, 0), (2, True, True, 4), (0, True, False, 3)])
@pytest.mark.parametrize("rows,K,C_,name", MANY)
def test_many_rows(kind, act, partial, bias, apart, rows, K, C_, name):
    run(rows, K, C_, kind, seed=7, bias=bias, act=act, partial=partial, stride=K + apart if apart else None)
    assert _lib.last_kernel() == "dense_f8_many_kernel" + name


def test_many_rows_two_at_once_and_replayed():
    for rows, K, C_, _ in MANY:
        x, w, other = U.operand(rows, C_, 1, 51), U.operand(K, C_, 128, 52), U.operand(rows, C_, 1, 53)
        ys = [torch.zeros(rows, K, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
        S.Dense(K, C_, x, w, U.buffer(ys[0]), batch=rows)
        S.Dense(K, C_, other, w, U.buffer(ys[1]), batch=rows)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(10):
            for s, v, y in zip(streams, (x, other), ys[2:]):
                S.Dense(K, C_, v, w, U.buffer(y), batch=rows, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(ys[2], ys[0]) and torch.equal(ys[3], ys[1])
        graph, buf = torch.cuda.CUDAGraph(), U.buffer(ys[2])
        with torch.cuda.graph(graph):
            S.Dense(K, C_, x, w, buf, batch=rows)
        x.t.copy_(other.t); x.scales.copy_(other.scales)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys[2], ys[1]) and _lib.device_status() == 0


@pytest.mark.parametrize("rows,K,C_,name", MANY)
def test_many_rows_of_nan_and_infinite_scales(rows, K, C_, name):
    x, w = U.operand(rows, C_, 1, 31), U.operand(K, C_, 128, 32)
    x.t.view(rows, C_).view(torch.uint8)[1, C_ - 1] = 0x7f
    x.scales.view(rows, -1)[2, 0] = torch.inf
    w.t.view(K, C_).view(torch.uint8)[131, 3] = 0xff
    y = torch.empty(rows, K, device="cuda")
    S.Dense(K, C_, x, w, U.buffer(y), batch=rows)
    assert _lib.last_kernel() == "dense_f8_many_kernel" + name
    want, size = U.dense(x, w)
    assert y[1].isnan().all() and y[:, 131].isnan().all()
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())
    fine = want.isfinite()
    assert ((y.double() - want).abs() <= U.dense_tolerance(want, size, C_, torch.float32))[fine].all()


def test_fp32_sums_are_as_near_as_fp32_sums_are():
    """Over many outputs the error is far below the bound that each of them has: no bits were lost between the tensor cores and the output.
    A sum of 128 terms with one truncation each is off by at most 128 * 2^-23 of the magnitudes, the mean over outputs by far less."""
    for rows in (8, 256, 2048):
        off, size = run(rows, 2048, 4096, "f32", seed=21, bias=False)
        assert (off.square().sum() / size.square().sum()).sqrt() < 2.0 ** -22


@pytest.mark.parametrize("rows", [3, 140])
def test_strided_operands(rows):
    """Rows of the operands and the output apart in memory, through the C ABI."""
    K, C_, apart = 200, 272, 320
    x, w = U.operand(rows, apart, 1, 1), U.operand(K, apart, 128, 2)
    nb = U.cdiv(C_, 128)
    xs, ws = (torch.rand(n, nb, device="cuda") + 0.5 for n in (rows, U.cdiv(K, 128)))
    y = torch.empty(rows, K, device="cuda")
    D = _lib.DenseLayer(rows, K, C_, _lib.TYPE_F32, apart, apart, 0, 0, 0, 0.0)
    _lib.check(_lib.lib().small_b200_dense_f8(C.byref(D), x.ptr(), xs.data_ptr(), w.ptr(), ws.data_ptr(), None, y.data_ptr(),
                                              torch.cuda.current_stream().cuda_stream))
    cut = lambda b, s, m: S.Float8Buffer(b.rows, C_, m, data=b.t.view(b.rows, apart)[:, :C_].contiguous(), scales=s)  # noqa: E731
    want, size = U.dense(cut(x, xs, 1), cut(w, ws, 128))
    assert ((y.double() - want).abs() <= U.dense_tolerance(want, size, C_, torch.float32)).all()


@pytest.mark.parametrize("rows", [4, 150])
def test_nan_and_infinite_scales_stay_in_their_rows(rows):
    K, C_ = 300, 400
    x, w = U.operand(rows, C_, 1, 31), U.operand(K, C_, 128, 32)
    codes = x.t.view(rows, C_).view(torch.uint8)
    codes[1, 399] = 0x7f                 # NaN
    x.scales.view(rows, -1)[2, 0] = torch.inf
    w.t.view(K, C_).view(torch.uint8)[131, 3] = 0xff
    y = torch.empty(rows, K, device="cuda")
    S.Dense(K, C_, x, w, U.buffer(y), batch=rows)
    want, size = U.dense(x, w)
    assert y[1].isnan().all() and y[:, 131].isnan().all()
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf()) and torch.equal(y[want.isinf()] > 0, want[want.isinf()] > 0)
    fine = want.isfinite()
    assert ((y.double() - want).abs() <= U.dense_tolerance(want, size, C_, torch.float32))[fine].all()


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("rows", [2, 150])
def test_activation_of_infinities(rows, act):
    x, w = U.operand(rows, 128, 1, 41), U.operand(16, 128, 128, 42)
    b = torch.tensor([torch.inf, -torch.inf, torch.nan] + [0.0] * 13, device="cuda")
    y = torch.empty(rows, 16, device="cuda")
    S.Dense_Bias_Activation(16, 128, x, w, S.FloatBuffer(data=b), U.buffer(y), activation=act, negative_slope=0.5, batch=rows)
    assert (y[:, 0] == torch.inf).all() and (y[:, 1] == (0 if act == 1 else -torch.inf)).all() and y[:, 2].isnan().all()


@pytest.mark.parametrize("rows", [1, 24, 160])
def test_two_streams_and_a_replayed_graph(rows):
    """Calls share nothing: two at once, and one captured and replayed on new data, give what one call alone gives."""
    K, C_ = 700, 4096
    x, w = U.operand(rows, C_, 1, 51), U.operand(K, C_, 128, 52)
    other = U.operand(rows, C_, 1, 53)
    alone = [torch.empty(rows, K, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    S.Dense(K, C_, x, w, U.buffer(alone[0]), batch=rows)
    S.Dense(K, C_, other, w, U.buffer(alone[1]), batch=rows)
    torch.cuda.synchronize()
    streams, ys = [torch.cuda.Stream() for _ in range(2)], [torch.zeros_like(alone[0]) for _ in range(2)]
    for _ in range(20):
        for s, v, y in zip(streams, (x, other), ys):
            S.Dense(K, C_, v, w, U.buffer(y), batch=rows, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(ys[0], alone[0]) and torch.equal(ys[1], alone[1])
    graph, y = torch.cuda.CUDAGraph(), torch.zeros_like(alone[0])
    buf = U.buffer(y)
    with torch.cuda.graph(graph):
        S.Dense(K, C_, x, w, buf, batch=rows)
    x.t.copy_(other.t); x.scales.copy_(other.scales)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, alone[1]) and _lib.device_status() == 0


def test_dense_bias_activation_of_fp32_buffers_is_the_convolution():
    rows, K, C_ = 9, 32, 48
    g = U.generator(60)
    x, f, b = (S.FloatBuffer(data=torch.randn(n, generator=g, device="cuda")) for n in (rows * C_, K * C_, K))
    one, two = S.FloatBuffer(rows * K), S.FloatBuffer(rows * K)
    S.Dense_Bias_Activation(K, C_, x, f, b, one, activation=S.ACT_RELU, batch=rows)
    S.Conv2D_Bias_ReLU(1, 1, 1, 0, 0, 0, 0, K, C_, 1, 1, x, f, b, two, batch=rows)
    assert torch.equal(one.t, two.t)
