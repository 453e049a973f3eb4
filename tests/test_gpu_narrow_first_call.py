"""The first call of each layer of narrow types in a process may be a captured one: whatever a launch sets up once a device takes part in no graph."""
import subprocess
import sys

import pytest
import torch

from smallframework_b200 import interface as S
from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
from smallframework_b200 import _lib, interface as S
from tests import narrow_util as U
rows, K, C = {rows}, {K}, 512
x, w = U.operand(rows, C, 1, 1), U.operand(K, C, 128, 2)
h = torch.randn(rows, C, device="cuda")
tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
y, q = S.FloatBuffer(rows * K), S.Float8Buffer(rows, C)
lp, ent, tv, ti = S.FloatBuffer(rows), S.FloatBuffer(rows), S.FloatBuffer(rows * 3), torch.empty(rows * 3, dtype=torch.int32, device="cuda")
y.t.zero_(); lp.t.zero_()
hb = S.FloatBuffer(data=h)
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    S.QuantizeBlocks(rows, C, hb, q)
    S.Dense(K, C, x, w, y, batch=rows)
    S.LogProbabilities(rows, K, y, tokens, lp, ent, tv, ti, top=3)
torch.cuda.synchronize()
assert (y.t == 0).all() and (lp.t == 0).all()
graph.replay()
torch.cuda.synchronize()
assert _lib.device_status() == 0
want, size = U.dense(x, w)
assert ((y.t.view(rows, K).double() - want).abs() <= U.dense_tolerance(want, size, C, torch.float32)).all()
assert torch.equal(ti.view(rows, 3).long(), U.logprobs(y.t.view(rows, K), tokens, 3)[3])
assert torch.equal(q.t.view(rows, C).double(), U.quantize(h, 1)[0])
print("captured")
"""


@pytest.mark.parametrize("rows,K", [(1, 40000), (5, 300), (2000, 2000)])
def test_first_call_is_captured(rows, K):
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(rows=rows, K=K)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_tensors_of_another_device_are_refused():
    x = S.FloatBuffer(data=torch.randn(4, 128, device="cuda:1"))
    with pytest.raises(ValueError):
        S.QuantizeBlocks(4, 128, x, S.Float8Buffer(4, 128, device="cuda:1"))
    with torch.cuda.device(1):
        out = S.Float8Buffer(4, 128)
        S.QuantizeBlocks(4, 128, x, out)
        torch.cuda.synchronize()


def test_python_refusals_on_the_device():
    """Buffers that are too small, of another type or not contiguous, before anything is launched."""
    x, w = S.Float8Buffer(3, 256), S.Float8Buffer(64, 256, 128)
    y = S.FloatBuffer(3 * 64)
    x.t.zero_(); w.t.zero_()
    S.Dense(64, 256, x, w, y, batch=3)
    cut = S.Float8Buffer(3, 256); cut.scales = torch.empty(5, device="cuda")
    for call in (lambda: S.Dense(64, 256, x, w, S.FloatBuffer(3 * 64 - 1), batch=3), lambda: S.Dense(64, 256, cut, w, y, batch=3),
                 lambda: S.Dense_Bias_Activation(64, 256, x, w, S.FloatBuffer(63), y, batch=3),
                 lambda: S.Dense_Bias_Activation(64, 256, x, w, S.HalfBuffer(64), y, batch=3),
                 lambda: S.Dense_Bias_Activation(64, 256, x, w, None, y, batch=3, output_stride=65),
                 lambda: S.Dense_Bias_Activation(64, 256, x, w, None, y, batch=3, output_stride=63),
                 lambda: S.Dense_Bias_Activation(64, 256, x, w, None, y, batch=3, activation=9),
                 lambda: S.QuantizeBlocks(3, 256, S.FloatBuffer(767), x), lambda: S.QuantizeBlocks(3, 256, S.QUInt8Buffer(768), x),
                 lambda: S.QuantizeBlocks(3, 256, S.FloatBuffer(768), cut), lambda: S.QuantizeBlocks(3, 256, S.FloatBuffer(768), x, input_stride=255),
                 lambda: S.LogProbabilities(3, 64, y, torch.zeros(3, dtype=torch.int16, device="cuda"), S.FloatBuffer(3)),
                 lambda: S.LogProbabilities(3, 64, y, torch.zeros(2, dtype=torch.int64, device="cuda"), S.FloatBuffer(3)),
                 lambda: S.LogProbabilities(3, 64, y, torch.zeros(6, dtype=torch.int64, device="cuda")[::2], S.FloatBuffer(3)),
                 lambda: S.LogProbabilities(3, 64, y, None, S.FloatBuffer(3)), lambda: S.LogProbabilities(3, 65, y, None, None, S.FloatBuffer(3)),
                 lambda: S.LogProbabilities(3, 64, y, None, None, None, S.FloatBuffer(5), top=2),
                 lambda: S.LogProbabilities(3, 64, y, None, None, None, None, torch.empty(6, dtype=torch.int64, device="cuda"), top=2),
                 lambda: S.LogProbabilities(3, 64, y, None, None, S.FloatBuffer(3), top=33)):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()
