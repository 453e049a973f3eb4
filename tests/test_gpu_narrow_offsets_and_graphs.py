"""The layers of narrow types where offsets pass 32 bits, and in captured graphs whose calls follow copies, other streams and one another."""
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U
from tests.test_gpu_logprobs import tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,K,stride", [(36000, 60001, 60008), (20, 500, 2 ** 27 + 8), (17, 130, 2 ** 27 + 1)])
def test_dense_outputs(rows, K, stride):
    assert (rows - 1) * stride + K > 2 ** 31
    x, w = U.operand(rows, 16, 1, 3), U.operand(K, 16, 128, 4)
    y = torch.zeros((rows - 1) * stride + K, device="cuda", dtype=torch.float16)
    S.Dense_Bias_Activation(K, 16, x, w, None, U.buffer(y), batch=rows, output_stride=stride)
    got = torch.as_strided(y, (rows, K), (stride, 1))
    for at in (0, rows // 2, rows - 3):
        some = S.Float8Buffer(3, 16, data=x.t.view(rows, 16)[at:at + 3].reshape(-1), scales=x.scales[at:at + 3])
        want, size = U.dense(some, w)
        tol = U.dense_tolerance(want, size, 16, torch.float16)
        assert (((got[at:at + 3].double() - want).abs() <= tol) | U.overflows(got[at:at + 3], want, tol, torch.float16)).all()
    assert (y[K:K + 5] == 0).all() if stride >= K + 5 else True


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,columns,stride", [(33000, 65552, 65552), (300, 528, 2 ** 23 + 8)])
def test_quantize_inputs(block_rows, rows, columns, stride):
    assert (rows - 1) * stride + columns > 2 ** 31
    x = torch.zeros((rows - 1) * stride + columns, device="cuda", dtype=torch.bfloat16)
    view = torch.as_strided(x, (rows, columns), (stride, 1))
    at = [0, rows // 128 * 128]
    assert at[1] * stride > 2 ** 31 - 1
    for a in at:
        view[a:a + 128].copy_(torch.randn(min(128, rows - a), columns, device="cuda", generator=U.generator(a)))
    q = S.Float8Buffer(rows, columns, block_rows)
    S.QuantizeBlocks(rows, columns, U.buffer(x), q, input_stride=stride)
    for a in at:
        want, scales = U.quantize(view[a:a + 128].contiguous(), block_rows)
        n = view[a:a + 128].shape[0]
        got = q.t.view(rows, columns)[a:a + n].double()
        per = q.scales.view(-1, U.cdiv(columns, 128))
        assert torch.equal(got, want.view(n, columns))
        assert torch.equal(per[a:a + n] if block_rows == 1 else per[a // 128:a // 128 + 1], scales.view(-1, per.shape[1]))


@pytest.mark.parametrize("rows,classes,stride", [(17000, 131072, 131072), (9, 5000, 2 ** 28 + 3), (700, 1000, 2 ** 22 + 1)])
def test_logits(rows, classes, stride):
    assert (rows - 1) * stride + classes > 2 ** 31
    x = torch.zeros((rows - 1) * stride + classes, device="cuda", dtype=torch.bfloat16)
    view = torch.as_strided(x, (rows, classes), (stride, 1))
    at = torch.tensor([0, rows // 2, rows - 1], device="cuda")
    view[at] = torch.randn(3, classes, device="cuda", generator=U.generator(1)).bfloat16() * 3
    tokens = torch.full((rows,), classes - 1, device="cuda")
    lp, h = S.FloatBuffer(rows), S.FloatBuffer(rows)
    tv, ti = S.FloatBuffer(rows * 8), torch.empty(rows * 8, dtype=torch.int32, device="cuda")
    S.LogProbabilities(rows, classes, U.buffer(x), tokens, lp, h, tv, ti, top=8, row_stride=stride)
    w_lp, w_h, w_tv, w_ti = U.logprobs(view[at].float(), tokens[at], 8)
    # 32 * classes: where a row is one warp's, a lane adds eight times as many terms as a thread of a CTA
    assert torch.equal(ti.view(rows, 8)[at].long(), w_ti)
    assert ((lp.t[at].double() - w_lp).abs() <= tolerance(x, w_lp, 32 * classes)[0]).all()
    assert ((tv.t.view(rows, 8)[at].double() - w_tv).abs() <= tolerance(x, w_tv, 32 * classes)[0]).all()
    assert ((h.t[at].double() - w_h).abs() <= tolerance(x, w_lp, 32 * classes)[1]).all()


@pytest.mark.parametrize("rows,K,C_", [(1, 640, 512), (24, 5000, 1024), (300, 4100, 528)])
def test_a_graph_with_copies_and_branches(rows, K, C_):
    """Calls that come after a copy, after another stream's call and after one another; replayed on new data."""
    g = U.generator(7)
    data = [torch.randn(rows, C_, device="cuda", generator=g).bfloat16() for _ in range(2)]
    weights = [torch.randn(K, C_, device="cuda", generator=g).half() for _ in range(2)]

    def buffers():
        return dict(x=torch.zeros(rows, C_, device="cuda", dtype=torch.bfloat16), w=torch.zeros(K, C_, device="cuda", dtype=torch.float16),
                    qx=S.Float8Buffer(rows, C_), qw=S.Float8Buffer(K, C_, 128), y=torch.zeros(rows, K, device="cuda"),
                    t=torch.zeros(rows, dtype=torch.long, device="cuda"), lp=torch.zeros(rows, device="cuda"), h=torch.zeros(rows, device="cuda"),
                    tv=torch.zeros(rows, 4, device="cuda"), ti=torch.zeros(rows, 4, dtype=torch.int32, device="cuda"))

    def steps(b, x, w, side):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        b["x"].copy_(x)
        S.QuantizeBlocks(rows, C_, U.buffer(b["x"].view(-1)), b["qx"])
        with torch.cuda.stream(side):
            b["w"].copy_(w)
            S.QuantizeBlocks(K, C_, U.buffer(b["w"].view(-1)), b["qw"])
        main.wait_stream(side)
        S.Dense(K, C_, b["qx"], b["qw"], U.buffer(b["y"].view(-1)), batch=rows)
        b["y"].mul_(0.5)
        S.LogProbabilities(rows, K, U.buffer(b["y"].view(-1)), b["t"], U.buffer(b["lp"]), U.buffer(b["h"]), U.buffer(b["tv"].view(-1)), b["ti"].view(-1), top=4)

    side = torch.cuda.Stream()
    want = []
    for x, w in zip(data, weights):
        b = buffers()
        steps(b, x, w, side)
        torch.cuda.synchronize()
        want.append({k: b[k].clone() for k in ("y", "lp", "h", "tv", "ti")})
    b, x, w = buffers(), data[0].clone(), weights[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(b, x, w, side)
    for n in (0, 1, 1, 0, 1):
        x.copy_(data[n]); w.copy_(weights[n])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(b[k], v) for k, v in want[n].items()) and _lib.device_status() == 0
