"""Refusals of the layers of narrow types: found on the host, before any CUDA call."""
import ctypes as C

import numpy as np
import pytest
import torch

from smallframework_b200 import _lib
from smallframework_b200 import interface as S

P = 1 << 20  # an address that is never followed: every call below is refused before a launch


def dense(code=None, **change):
    D = dict(rows=4, K=100, C=128, out_type=_lib.TYPE_BF16, in_stride=0, filt_stride=0, out_stride=0, accumulate=0, act=0, slope=0.0)
    p = {k: change.pop(k, P) for k in ("inp", "in_scales", "filt", "filt_scales", "bias", "out")}
    D.update(change)
    rc = _lib.lib().small_b200_dense_f8(C.byref(_lib.DenseLayer(**D)), p["inp"], p["in_scales"], p["filt"], p["filt_scales"], p["bias"], p["out"], None)
    return rc, _lib.lib().small_b200_last_error().decode()


@pytest.mark.parametrize("change,words", [
    (dict(C=0), "in_channels"), (dict(C=-16), "in_channels"), (dict(C=100), "in_channels"), (dict(K=0), "out_channels"), (dict(K=-1), "out_channels"),
    (dict(out_type=3), "output type"), (dict(out_type=-1), "output type"), (dict(act=7), "activation"), (dict(rows=-1), "bad shape"),
    (dict(in_stride=112), "bad shape"), (dict(in_stride=130), "bad shape"), (dict(filt_stride=64), "bad shape"), (dict(out_stride=99), "bad shape"),
    (dict(in_stride=-128), "bad shape"), (dict(in_stride=1 << 40), "bad shape"),
    (dict(inp=None), "null"), (dict(in_scales=None), "null"), (dict(filt=None), "null"), (dict(filt_scales=None), "null"), (dict(out=None), "null"),
    (dict(inp=P + 8), "misaligned"), (dict(filt=P + 1), "misaligned"), (dict(in_scales=P + 2), "misaligned"), (dict(bias=P + 2), "misaligned"),
    (dict(out=P + 1), "misaligned"), (dict(out=P + 2, out_type=_lib.TYPE_F32), "misaligned"), (dict(rows=0x7fffffff, K=0x7fffffff), "too many tiles"),
])
def test_dense_refuses(change, words):
    rc, said = dense(**change)
    assert rc == _lib.INVALID_ARGUMENT and words in said and said.startswith("Dense<float8> ERROR")


def test_no_rows_is_no_work():
    assert dense(rows=0, inp=None, in_scales=None, filt=None, filt_scales=None, bias=None, out=None)[0] == _lib.OK
    l = _lib.lib()
    assert l.small_b200_quantize_blocks_f8(0, 128, 1, 0, None, 0, None, None, None) == _lib.OK
    assert l.small_b200_logprobs(0, 10, 0, None, 0, 4, None, None, None, 0, None, None, None) == _lib.OK
    assert l.small_b200_logprobs(3, 10, 0, P, 0, 4, None, None, None, 5, None, None, None) == _lib.OK  # nothing asked for
    assert dense(rows=0)[0] == _lib.OK
    assert l.small_b200_dense_f8(None, P, P, P, P, P, P, None) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("args,words", [
    ((4, 0, 1, 0, P, 0, P, P), "in_channels"), ((4, 24, 1, 0, P, 0, P, P), "in_channels"), ((-1, 16, 1, 0, P, 0, P, P), "bad shape"),
    ((4, 16, 64, 0, P, 0, P, P), "bad shape"), ((4, 16, 0, 0, P, 0, P, P), "bad shape"), ((4, 32, 1, 0, P, 16, P, P), "bad shape"),
    ((4, 16, 1, 5, P, 0, P, P), "input type"), ((4, 16, 1, 0, None, 0, P, P), "null"), ((4, 16, 1, 0, P, 0, None, P), "null"),
    ((4, 16, 1, 0, P, 0, P, None), "null"), ((4, 16, 1, 0, P + 2, 0, P, P), "misaligned"), ((4, 16, 1, 1, P + 1, 0, P, P), "misaligned"),
    ((4, 16, 1, 0, P, 0, P + 8, P), "misaligned"), ((4, 16, 1, 0, P, 0, P, P + 2), "misaligned"), ((0x7fffffff, 256, 1, 0, P, 0, P, P), "too many blocks"),
])
def test_quantize_refuses(args, words):
    assert _lib.lib().small_b200_quantize_blocks_f8(*args, None) == _lib.INVALID_ARGUMENT
    said = _lib.lib().small_b200_last_error().decode()
    assert words in said and said.startswith("QuantizeBlocks<float8> ERROR")


@pytest.mark.parametrize("change,words", [
    (dict(rows=-1), "bad shape"), (dict(classes=0), "bad shape"), (dict(stride=99), "bad shape"), (dict(kind=9), "input type"),
    (dict(token_bytes=2), "tokens"), (dict(top=-1), "top unsupported"), (dict(top=33), "top unsupported"), (dict(classes=4, top=5), "top unsupported"),
    (dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(logits=P + 2), "misaligned"), (dict(logits=P + 1, kind=1), "misaligned"),
    (dict(tokens=P + 4, token_bytes=8), "misaligned"), (dict(lp=P + 1), "misaligned"), (dict(h=P + 2), "misaligned"), (dict(tv=P + 2), "misaligned"),
    (dict(ti=P + 2), "misaligned"),
])
def test_logprobs_refuse(change, words):
    a = dict(rows=3, classes=100, kind=0, logits=P, stride=0, token_bytes=4, tokens=P, lp=P, h=P, top=4, tv=P, ti=P)
    a.update(change)
    assert _lib.lib().small_b200_logprobs(*a.values(), None) == _lib.INVALID_ARGUMENT
    said = _lib.lib().small_b200_last_error().decode()
    assert words in said and said.startswith("LogProbabilities ERROR")


def test_python_refuses_buffers_that_do_not_fit():
    cpu = dict(device="cpu")
    x, w = S.Float8Buffer(2, 256, **cpu), S.Float8Buffer(100, 256, 128, **cpu)
    y = S.BFloat16Buffer(200, **cpu)
    for call in (lambda: S.Float8Buffer(2, 256, 64), lambda: S.Float8Buffer(2, 256, scales=torch.ones(3), **cpu),
                 lambda: S.Float8Buffer(2, 256, data=np.zeros(500, np.uint8), **cpu),
                 lambda: S.Dense(100, 256, y, w, y, batch=2), lambda: S.Dense(100, 256, w, w, y, batch=2), lambda: S.Dense(100, 256, x, x, y, batch=2),
                 lambda: S.Dense(99, 256, x, w, y, batch=2), lambda: S.Dense(100, 128, x, w, y, batch=2), lambda: S.Dense(100, 256, x, w, y, batch=3),
                 lambda: S.Dense(100, 256, x, w, x, batch=2), lambda: S.Dense(100, 256, x, w, S.QUInt8Buffer(200, **cpu), batch=2),
                 lambda: S.QuantizeBlocks(2, 256, y, y), lambda: S.QuantizeBlocks(3, 256, S.FloatBuffer(768, **cpu), x),
                 lambda: S.QuantizeBlocks(1 << 32, 256, y, x), lambda: S.LogProbabilities(1 << 32, 10, y, None, None, y),
                 lambda: S.Dense_Bias_Activation(16, 16, S.FloatBuffer(16, **cpu), S.FloatBuffer(256, **cpu), None, S.FloatBuffer(16, **cpu), output_stride=32)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: S.Dense(100, 256, x, w, y, batch=2), lambda: S.QuantizeBlocks(2, 256, S.FloatBuffer(512, **cpu), x),
                 lambda: S.LogProbabilities(2, 10, S.HalfBuffer(20, **cpu), None, None, S.FloatBuffer(2, **cpu))):
        with pytest.raises(_lib.SmallB200Error):  # no CPU path
            call()


def test_other_layers_refuse_narrow_buffers():
    """A layer that counts elements of four bytes must not be handed two-byte ones."""
    n = S.BFloat16Buffer(512, device="cpu")
    for call in (lambda: S.ReLUActivation(16, 4, 4, n, n), lambda: S.Conv2D(1, 1, 1, 0, 0, 0, 0, 16, 16, 4, 4, n, n, n),
                 lambda: S.SoftMax(16, 4, 4, n, n), lambda: S.Dense(16, 16, n, n, n)):
        with pytest.raises(ValueError):
            call()


def test_numpy_data_keeps_its_values():
    assert np.array_equal(S.BFloat16Buffer(data=np.float32([1.5, -2, 300]), device="cpu").numpy(), np.float32([1.5, -2, 300]))
    assert S.HalfBuffer(data=np.float32([1.5]), device="cpu").t.dtype == torch.float16
    b = S.Float8Buffer(1, 4, data=np.uint8([0x38, 0xb8, 0x7e, 0x01]), scales=np.float32([2]), device="cpu")  # 1, -1, 448, 2^-9
    assert b.dequantized().tolist() == [[2.0, -2.0, 896.0, 2.0 ** -8]]
