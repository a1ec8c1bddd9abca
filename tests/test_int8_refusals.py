"""Refusals of the int8 layer's and the row rotation's entry points: the checks come
before any device call, so these need no GPU."""
import ctypes
import math

import numpy as np
import pytest

import mini_llama_b200 as mlb
from mini_llama_b200 import _lib
from tests import int8_ref

P = 1 << 24  # never dereferenced: the checks come first


def err(rc, text, code=-1):
    assert rc == code, (rc, _lib.lib().mlb_last_error())
    assert text.encode() in _lib.lib().mlb_last_error(), _lib.lib().mlb_last_error()


def passes(rc):
    """Refused for the device alone (there is none here), or done."""
    assert rc != 0 and b"cuda" in _lib.lib().mlb_last_error().lower(), _lib.lib().mlb_last_error()


def no_gpu():
    try:
        return mlb.CudaDeviceCount() == 0
    except mlb.MlbError:
        return True


needs_no_gpu = pytest.mark.skipif(not no_gpu(), reason="these calls would run")


def quantize(**kw):
    a = dict(act=0, x=P, xs=100, rows=4, n=100, codes=P + (1 << 20), cs=112, scales=P + (2 << 20))
    a.update(kw)
    return _lib.lib().mlb_int8_quantize(*a.values(), 0, None)


def test_quantize_is_refused():
    err(quantize(act=2), "unknown activation type 2")
    err(quantize(rows=-1), "negative row count")
    err(quantize(n=0), "at least one element")
    err(quantize(n=(1 << 28) + 1), "more than 2^28")
    err(quantize(x=None), "null x")
    err(quantize(x=P + 2), "x is unaligned")
    err(quantize(act=1, x=P + 1), "x is unaligned")
    err(quantize(xs=99), "row stride of x is smaller")
    err(quantize(codes=None), "null codes")
    err(quantize(codes=P + (1 << 20) + 8), "rows of codes must be 16-byte aligned")
    err(quantize(cs=104), "rows of codes must be 16-byte aligned")
    err(quantize(cs=96), "row stride of codes is smaller")
    err(quantize(scales=None), "null scales")
    err(quantize(scales=P + (2 << 20) + 2), "scales are unaligned")
    err(quantize(codes=P), "codes must not overlap x")
    err(quantize(codes=P + 1584), "codes must not overlap x")
    err(quantize(scales=P + 1596), "scales must not overlap x")
    err(quantize(scales=P + (1 << 20) + 112), "codes must not overlap scales")


def norm(**kw):
    a = dict(act=0, x=P, xs=128, r=P + (1 << 20), rs=128, w=P + (2 << 20), rows=4, n=128, eps=1e-5,
             sum=P + (3 << 20), ss=128, codes=P + (4 << 20), cs=128, scales=P + (5 << 20))
    a.update(kw)
    return _lib.lib().mlb_rmsnorm_int8(*a.values(), 0, None)


def test_norm_is_refused():
    err(norm(act=9), "unknown activation type 9")
    for eps in (-1e-9, math.nan, math.inf):
        err(norm(eps=eps), "eps must be finite and not negative")
    err(norm(w=None), "null weights")
    err(norm(w=P + (2 << 20) + 1), "weights are unaligned")
    err(norm(x=None), "null x")
    err(norm(rs=127), "row stride of residual is smaller")
    err(norm(sum=None), "null sum")
    err(norm(ss=100), "row stride of sum is smaller")
    err(norm(r=None), "a sum without a residual")
    err(norm(sum=P + 512), "sum must not overlap x")
    err(norm(sum=P, ss=132), "sum must not overlap x")
    err(norm(sum=P + (1 << 20) + 4), "sum must not overlap residual")
    err(norm(sum=P + (2 << 20)), "sum must not overlap weights")
    err(norm(codes=P + (3 << 20)), "codes must not overlap sum")
    err(norm(codes=P + (2 << 20)), "codes must not overlap weights")
    err(norm(scales=P + (1 << 20)), "scales must not overlap residual")
    err(norm(codes=P + 1024), "codes must not overlap x")


def silu(**kw):
    a = dict(act=0, g=P, gs=256, u=P + 512, us=256, rows=4, n=128, codes=P + (4 << 20), cs=128,
             scales=P + (5 << 20))
    a.update(kw)
    return _lib.lib().mlb_silu_mul_int8(*a.values(), 0, None)


def test_silu_is_refused():
    err(silu(act=-1), "unknown activation type -1")
    err(silu(g=None), "null gate")
    err(silu(u=None), "null up")
    err(silu(us=127), "row stride of up is smaller")
    err(silu(codes=P), "codes must not overlap gate")
    err(silu(codes=P + 512), "codes must not overlap up")
    err(silu(scales=P + 3 * 1024 + 496), "scales must not overlap gate")


def dequantize(**kw):
    a = dict(codes=P, cs=112, scales=P + (1 << 20), rows=4, n=100, act=0, out=P + (2 << 20), os=100)
    a.update(kw)
    return _lib.lib().mlb_int8_dequantize(*a.values(), 0, None)


def test_dequantize_is_refused():
    err(dequantize(act=5), "unknown activation type 5")
    err(dequantize(out=None), "null out")
    err(dequantize(os=99), "row stride of out is smaller")
    err(dequantize(out=P), "out must not overlap codes")
    err(dequantize(out=P + (1 << 20) + 12), "out must not overlap scales")
    err(dequantize(cs=100), "rows of codes must be 16-byte aligned")


def linear(**kw):
    a = dict(x=P, xs=128, sx=P + (1 << 20), rows=4, k=100, w=P + (2 << 20), ws=112, sw=P + (3 << 20),
             n=60, bias=P + (4 << 20), act=0, out=P + (5 << 20), os=60)
    a.update(kw)
    return _lib.lib().mlb_int8_linear(*a.values(), 0, None)


def test_linear_is_refused():
    err(linear(act=4), "unknown activation type 4")
    err(linear(rows=-1), "negative row count")
    err(linear(k=0), "in_features must be 1 to 131071")
    err(linear(k=131072, xs=131072, ws=131072), "in_features must be 1 to 131071")
    err(linear(n=0), "out_features must be 1 to 2^28")
    for name, at in (("x", "xs"), ("w", "ws")):
        err(linear(**{name: None}), f"null {name}")
        err(linear(**{name: P + 8}), f"rows of {name} must be 16-byte aligned")
        err(linear(**{at: 104}), f"rows of {name} must be 16-byte aligned")
        err(linear(**{at: 96}), f"row stride of {name} is smaller")
        err(linear(**{at: 1 << 40}), f"row stride of {name} must be below 2^40")
    err(linear(sx=None), "null x_scale")
    err(linear(sw=P + 2), "w_scale is unaligned")
    err(linear(bias=P + 3), "bias is unaligned")
    err(linear(out=None), "null out")
    err(linear(out=P + (5 << 20) + 2), "out is unaligned")
    err(linear(os=59), "row stride of out is smaller")
    err(linear(out=P + 480), "out must not overlap x")
    err(linear(out=P + (2 << 20) + 112 * 59 + 96), "out must not overlap w")
    err(linear(out=P + (1 << 20)), "out must not overlap x_scale")
    err(linear(out=P + (3 << 20)), "out must not overlap w_scale")
    err(linear(out=P + (4 << 20)), "out must not overlap bias")
    f = _lib.lib().mlb_int8_linear_wait_selftest
    c = ctypes.c_int()
    err(f(0, 8, 0.0, c, c, c), "limit_ms must be in (0, 1000]")
    err(f(0, 8, math.nan, c, c, c), "limit_ms must be in (0, 1000]")
    err(f(0, 0, 1.0, c, c, c), "rows must be 1 to 1024")
    err(f(0, 8, 1.0, None, c, c), "null output")
    err(_lib.lib().mlb_int8_linear_status(0, None, c), "null output")


def rope(**kw):
    a = dict(act=0, q=P, qs=256, heads=4, k=P + (1 << 20), ks=128, kv=2, dim=64, rot=32,
             pos=P + (2 << 20), f=P + (3 << 20), gain=1.0, kind=0, rows=3, qo=P + (4 << 20), qos=256,
             ko=P + (5 << 20), kos=128)
    a.update(kw)
    return _lib.lib().mlb_rope_rows(*a.values(), 0, None)


def test_rope_is_refused():
    err(rope(act=3), "unknown activation type 3")
    err(rope(kind=2), "unknown rope type 2")
    err(rope(kind=-1), "unknown rope type -1")
    err(rope(rows=-1), "negative row count")
    err(rope(heads=-1), "negative head count")
    for dim in (0, 63, 1026):
        err(rope(dim=dim), "head_dim must be even, 2 to 1024")
    for rot in (0, 31, 66):
        err(rope(rot=rot), "rotary_dim must be even, 2 to head_dim")
    err(rope(gain=math.nan), "amplitude must be finite")
    err(rope(pos=None), "null positions or frequencies")
    err(rope(f=P + 4), "positions or frequencies are unaligned")
    err(rope(q=None), "null q")
    err(rope(ko=None), "null k_out")
    err(rope(qs=255), "row stride of q is smaller")
    err(rope(kos=127), "row stride of k_out is smaller")
    err(rope(k=P + (1 << 20) + 2), "k is unaligned")
    err(rope(qo=P + 16), "q_out must not overlap q")
    err(rope(qo=P, qos=512), "q_out must not overlap q")
    err(rope(qo=P + (1 << 20) + 512), "q_out must not overlap k")
    err(rope(qo=P + (5 << 20)), "q_out must not overlap k_out")
    err(rope(ko=P), "k_out must not overlap q")
    err(rope(ko=P + (2 << 20)), "k_out must not overlap positions")
    err(rope(qo=P + (3 << 20)), "q_out must not overlap frequencies")


@needs_no_gpu
def test_calls_that_are_taken():
    """In place, side by side in one buffer, one row of any stride."""
    passes(rope(qo=P, ko=P + (1 << 20)))
    passes(rope(qs=384, qo=P, qos=384, k=P + 1024, ks=384, ko=P + 1024, kos=384))
    passes(rope(rows=1, qs=1 << 50, qo=P, qos=1 << 40))
    passes(rope(heads=0, q=None, qo=None))
    passes(norm(sum=P))
    passes(norm(sum=P + (1 << 20)))
    passes(norm(r=P, sum=P))
    passes(norm(rows=1, sum=P, ss=1000))
    passes(norm(r=None, sum=None))
    passes(silu())
    passes(linear(bias=None))
    passes(linear(rows=0, x=None))
    passes(quantize(rows=0, x=None))


def frequencies(rot=64, theta=1e4, kind=0, factor=8.0, trained=8192.0, low=1.0, high=4.0, fast=32.0,
                slow=1.0):
    f, a = np.zeros(512), ctypes.c_double(-1)
    rc = _lib.lib().mlb_rope_frequencies(rot, theta, kind, factor, trained, low, high, fast, slow,
                                         f.ctypes.data_as(ctypes.POINTER(ctypes.c_double)),
                                         ctypes.byref(a))
    return rc, f[:max(rot, 0) // 2], a.value


def test_frequencies_are_refused():
    for rot in (0, 7, 1026, -2):
        err(frequencies(rot)[0], "rotary_dim must be even, 2 to 1024")
    for theta in (1.0, -1.0, math.nan, math.inf):
        err(frequencies(theta=theta)[0], "theta must be finite and above 1")
    err(frequencies(kind=4)[0], "unknown scaling 4")
    err(frequencies(kind=1, factor=0.0)[0], "factor must be finite and positive")
    err(frequencies(kind=2, trained=0.0)[0], "original_len must be finite and positive")
    err(frequencies(kind=2, low=4.0)[0], "low_freq_factor must be positive and below")
    err(frequencies(kind=3, slow=33.0)[0], "beta_slow must be positive and at most")
    a = ctypes.c_double()
    err(_lib.lib().mlb_rope_frequencies(64, 1e4, 0, 1, 1, 1, 1, 1, 1, None, ctypes.byref(a)),
        "null output")


@pytest.mark.parametrize("kind,name", list(enumerate(["none", "linear", "llama3", "yarn"])))
@pytest.mark.parametrize("rot,theta,trained", [(128, 500000.0, 8192.0), (64, 1e4, 2048.0),
                                               (2, 1e4, 4096.0), (48, 1e6, 32768.0),
                                               (10, 1e4, 100.0), (128, 1e4, 4.0)])
def test_frequencies(kind, name, rot, theta, trained):
    pytest.importorskip("torch")
    for factor in (8.0, 0.5, 1.0):
        rc, f, gain = frequencies(rot, theta, kind, factor, trained)
        assert rc == 0
        want, want_gain = int8_ref.frequencies(rot, theta, name, factor, trained)
        # powers and quotients of a few 64-bit roundings
        assert np.allclose(f, want.numpy(), rtol=1e-13, atol=0)
        assert math.isclose(gain, want_gain, rel_tol=1e-15)


def test_python_forms_refuse_before_the_device():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 32)
    q = torch.zeros(2, 32, dtype=torch.int8)
    for call in (lambda: mlb.CudaInt8QuantizeDeviceInput(x.half()),
                 lambda: mlb.CudaSiluMulInt8DeviceInput(x.double(), x),
                 lambda: mlb.CudaInt8LinearDeviceInput(q, x, q, x, out_dtype=torch.float16)):
        with pytest.raises(mlb.MlbError, match="expected float32 or bfloat16"):
            call()
    for call in (lambda: mlb.CudaInt8QuantizeDeviceInput(x),
                 lambda: mlb.CudaRmsNormInt8DeviceWeight(x, x[0], 1e-5),
                 lambda: mlb.CudaSiluMulInt8DeviceInput(x, x),
                 lambda: mlb.CudaInt8DequantizeDeviceInput(q, x[0]),
                 lambda: mlb.CudaInt8LinearDeviceInput(q, x[0], q, x[0])):
        with pytest.raises(mlb.MlbError, match="must be on a CUDA device"):
            call()
    with pytest.raises(mlb.MlbError, match="expected x"):
        mlb.CudaInt8QuantizeDeviceInput(x[None])
    with pytest.raises(mlb.MlbError, match="expected int8"):
        mlb.CudaInt8LinearDeviceInput(x, x[0], q, x[0])
    with pytest.raises(mlb.MlbError, match="rotary_dim must be even"):
        mlb.RopeTable(63)


@pytest.mark.parametrize("there", [True, False])
def test_a_build_without_torch_leaves_out_its_calls(monkeypatch, there):
    from mini_llama_b200 import build

    made = []
    for name in ("build_synth", "build_cuda", "build_calls"):
        monkeypatch.setattr(build, name, lambda *a, name=name: made.append(name))
    monkeypatch.setattr(build.importlib.util, "find_spec",
                        build.importlib.util.find_spec if there else lambda name: None)
    build.build()
    assert made == ["build_synth", "build_cuda"] + ["build_calls"] * there
    if not there:
        monkeypatch.undo()
        monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
        with pytest.raises(RuntimeError, match="need torch"):
            build.build_calls(force=True)
