"""Ways to call the layers of narrow types that their documents allow: threads that share a stream, fewer rows than a buffer has, a stream by its number."""
import threading

import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S
from tests import narrow_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,K,C_", [(2, 2 * 148 * 128 + 645, 2048), (24, 640, 4096), (300, 4109, 272), (2300, 2310, 400)])
def test_threads_on_one_stream(rows, K, C_):
    """Each thread's quantisation, layer (one launch or two) and log-probabilities stand between the others' in the stream, in any order."""
    w, stream = U.operand(K, C_, 128, 1, spread_of_scales=0.5), torch.cuda.Stream()
    jobs = []
    for n in range(4):
        hidden = (torch.randn(rows, C_, generator=U.generator(n), device="cuda")).bfloat16()
        jobs.append(dict(h=U.buffer(hidden), q=S.Float8Buffer(rows, C_), y=torch.zeros(rows * K, device="cuda"), lp=torch.zeros(rows, device="cuda"),
                         ti=torch.zeros(rows * 5, dtype=torch.int32, device="cuda"), t=torch.full((rows,), n, device="cuda")))

    def once(j):
        S.QuantizeBlocks(rows, C_, j["h"], j["q"], stream=stream)
        S.Dense(K, C_, j["q"], w, U.buffer(j["y"]), batch=rows, stream=stream)
        S.LogProbabilities(rows, K, U.buffer(j["y"]), j["t"], U.buffer(j["lp"]), None, None, j["ti"], top=5, stream=stream)

    torch.cuda.synchronize()
    for j in jobs:
        once(j)
    torch.cuda.synchronize()
    want = [[j[k].clone() for k in ("y", "lp", "ti")] for j in jobs]
    failed = []

    def work(j):
        try:
            for _ in range(40):
                once(j)
        except Exception as e:
            failed.append(e)

    for j in jobs:
        j["y"].zero_(); j["lp"].zero_(); j["ti"].zero_(); j["q"].scales.zero_()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and _lib.device_status() == 0
    for j, v in zip(jobs, want):
        assert all(torch.equal(j[k], a) for k, a in zip(("y", "lp", "ti"), v))


@pytest.mark.parametrize("rows,of", [(1, 5), (17, 40), (300, 301), (2, 3000)])
def test_fewer_rows_than_the_buffers_have(rows, of):
    K, C_ = 333, 272
    x, w = U.operand(of, C_, 1, 1), U.operand(K, C_, 128, 2)
    y = torch.full((of, K), 7.0, device="cuda")
    S.Dense(K, C_, x, w, U.buffer(y), batch=rows)
    first = S.Float8Buffer(rows, C_, data=x.t[:rows * C_], scales=x.scales[:rows * U.cdiv(C_, 128)])
    want, size = U.dense(first, w)
    assert ((y[:rows].double() - want).abs() <= U.dense_tolerance(want, size, C_, torch.float32)).all()
    assert (y[rows:] == 7).all()
    lp, ti = torch.full((of,), 7.0, device="cuda"), torch.full((of * 3,), 7, dtype=torch.int32, device="cuda")
    S.LogProbabilities(rows, K, U.buffer(y), torch.zeros(of, dtype=torch.int64, device="cuda"), U.buffer(lp), None, None, ti, top=3)
    assert (lp[rows:] == 7).all() and (ti[rows * 3:] == 7).all() and (lp[:rows] <= 0).all()


def test_a_stream_by_its_number():
    rows, K, C_ = 4, 640, 512
    s = torch.cuda.Stream()
    x, w, q = torch.randn(rows, C_, device="cuda"), U.operand(K, C_, 128, 2), S.Float8Buffer(rows, C_)
    y, z = torch.zeros(rows, K, device="cuda"), torch.zeros(rows, K, device="cuda")
    torch.cuda.synchronize()
    S.QuantizeBlocks(rows, C_, U.buffer(x), q, stream=s.cuda_stream)
    S.Dense(K, C_, q, w, U.buffer(y), batch=rows, stream=s.cuda_stream)
    s.synchronize()
    with torch.cuda.stream(s):
        S.Dense(K, C_, q, w, U.buffer(z), batch=rows)
    s.synchronize()
    assert torch.equal(y, z) and torch.equal(q.t.view(rows, C_).double(), U.quantize(x, 1)[0])
