"""Refusals of the paged attention's entry points that need no GPU: the checks come
before any device call."""
import ctypes
import random

import pytest

import mini_llama_b200 as mlb
from mini_llama_b200 import _lib


def err(rc, text, code=-1):
    assert rc == code, (rc, _lib.lib().mlb_last_error())
    assert text.encode() in _lib.lib().mlb_last_error(), _lib.lib().mlb_last_error()


P = 1 << 20  # never dereferenced: a call that passes these checks is refused for its workspace


def attend(q=0, out=0, qs=256, outs=256, rows=3, act=0):
    n = _lib.lib().mlb_paged_attention(
        P, 2, 4, 16, 2, 64, 0, act, P + q, qs, 4, rows, 1, P, P, P, 64, 0.1, P + out, outs, None, 0,
        0, None)
    assert n != 0
    return b"must not overlap" in _lib.lib().mlb_last_error()


def shares(q=0, out=0, qs=256, outs=256, rows=3, act=0):
    """Whether a byte belongs to a row of both (4 heads of 64), row by row."""
    es = 2 if act else 4
    n = 256 * es
    return any(abs(q + i * qs * es - out - j * outs * es) < n
               for i in range(rows) for j in range(rows))


@pytest.mark.parametrize("call", [
    dict(out=0), dict(out=16), dict(q=16), dict(out=1008), dict(out=1024), dict(out=2048),
    dict(q=3056), dict(out=2048 + 1008), dict(out=512, qs=512), dict(out=2048, qs=512, rows=2),
    dict(out=1024, outs=512), dict(q=512, qs=512, outs=384), dict(q=8192, outs=2048),
    dict(act=1, out=496), dict(act=1, out=1408, qs=512, outs=512, rows=4),
    dict(q=2048 * 100 + 1008, qs=260, outs=512, rows=300)])
def test_attention_refuses_outputs_over_queries(call):
    assert shares(**call) and attend(**call)


@pytest.mark.parametrize("call", [
    dict(out=4096, rows=4), dict(q=4096, rows=4), dict(out=1024, qs=512, outs=512), dict(q=1024, qs=512, outs=512),
    dict(out=1024, rows=1), dict(out=1024, qs=512, outs=768, rows=2), dict(q=4096, outs=2048),
    dict(act=1, out=512, qs=512, outs=512), dict(act=1, out=512, rows=1, qs=512, outs=264),
    dict(act=1, out=1536, qs=512, outs=512, rows=4),
    dict(out=1024 + 512, qs=768, outs=768, rows=300), dict(q=P, qs=1 << 40, outs=1 << 41)])
def test_attention_takes_rows_side_by_side(call):
    assert not shares(**call) and not attend(**call)


@pytest.mark.parametrize("stride", [1 << 60, 1 << 61, 1 << 62, (1 << 63) - 8])
def test_strides_whose_bytes_pass_64_bits(stride):
    for act in (0, 1):
        for rows in (1, 3):
            assert not attend(out=2048, qs=stride, act=act, rows=rows)
            assert not attend(q=2048, outs=stride, act=act, rows=rows)
            assert attend(qs=stride, outs=stride, act=act, rows=rows)
            assert attend(q=16, qs=stride, act=act, rows=rows)


def test_any_two_sets_of_rows():
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(3000):
        act = rng.randrange(2)
        unit = 8 if act else 4  # elements in 16 bytes
        qs = 256 + unit * rng.randrange(0, 200)
        call = dict(act=act, qs=qs, outs=rng.choice([qs, 256 + unit * rng.randrange(0, 200)]),
                    rows=rng.randrange(1, 12), q=16 * rng.randrange(0, 600),
                    out=16 * rng.randrange(0, 600))
        want = shares(**call)
        assert attend(**call) == want, call
        seen[want] += 1
    assert min(seen) > 300


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38, float("nan"), float("-inf")])
def test_scales_past_the_exponent_range_are_refused(scale):
    """Scores are taken in powers of two: scale log2(e) has to be a number."""
    n = _lib.lib().mlb_paged_attention(P, 2, 4, 16, 2, 64, 0, 0, P, 256, 4, 3, 1, P, P, P, 64, scale,
                                       P + 4096, 256, None, 0, 0, None)
    assert n == -1 and b"scale must be finite" in _lib.lib().mlb_last_error()


def append(q=0, qo=1 << 16, k=1 << 17, v=1 << 18, qs=256, qos=256, ks=128, vs=128, rows=3):
    n = _lib.lib().mlb_paged_kv_append(
        P, 2, 4, 16, 2, 64, 0, 0, P + k, ks, P + v, vs, P + q, qs, 4, P + qo, qos, rows, 1, P, P, P,
        2, 1e4, 0, 0, None)
    assert n == -1
    return _lib.lib().mlb_last_error().decode()


# every one of these is refused: a call that is not would launch on addresses of no one
@pytest.mark.parametrize("call", [
    dict(qo=16), dict(qo=1024), dict(q=3056, qo=0), dict(qo=0, qos=512), dict(qo=0, qs=512),
    dict(qo=512, qs=512, qos=512)])
def test_append_refuses_queries_out_over_queries(call):
    assert "q_out must be q itself or not overlap it" in append(**call)


@pytest.mark.parametrize("call", [
    dict(qo=1 << 17), dict(k=4096, qo=4096 + 1520), dict(q=4096, qo=4096, v=4096),
    dict(k=8192, ks=640, qo=8192 + 256, qos=640), dict(k=1 << 14, ks=512, v=1 << 15, qo=(1 << 15) - 512)])
def test_append_refuses_queries_out_over_keys_or_values(call):
    assert "q_out must not overlap k or v" in append(**call)


def test_read_refuses_values_over_keys():
    for k, v in ((0, 0), (0, 1520), (1024, 0)):  # three rows of 512 bytes
        n = _lib.lib().mlb_paged_kv_read(P, 2, 4, 16, 2, 64, 0, 3, 1, P, P, P, 2, P + k, P + v, 0,
                                         None)
        assert n == -1 and b"k_out and v_out must not overlap" in _lib.lib().mlb_last_error()


def test_wait_selftest_refuses_bad_arguments():
    f = _lib.lib().mlb_paged_attention_wait_selftest
    a, b, c = (ctypes.byref(ctypes.c_int()) for _ in range(3))
    err(f(0, 0, 1.0, None, b, c), "null output")
    err(f(0, 0, 1.0, a, b, None), "null output")
    err(f(0, 2, 1.0, a, b, c), "unknown activation type 2")
    for limit in (0.0, -1.0, 1001.0, float("nan")):
        with pytest.raises(mlb.MlbError, match="limit_ms"):
            mlb.paged_attention_wait_selftest(limit_ms=limit)


def test_reset_that_fails_leaves_an_empty_cache(monkeypatch):
    """Not the old pool under the new shape, which every later call would overrun."""
    torch = pytest.importorskip("torch")
    made = []

    def zeros(shape, **kw):
        if made:
            raise RuntimeError("out of memory")
        made.append(shape)
        return torch.empty(1)

    monkeypatch.setattr(torch, "zeros", zeros)
    cache = mlb.CudaPagedKvCache(1, 2, 16, 2, 64)
    assert not cache.empty() and cache.n_pages() == 2
    with pytest.raises(mlb.MlbError, match="multiple of 16"):
        cache.Reset(1, 4, 24, 2, 64)
    assert cache.n_pages() == 2  # refused before anything changed
    with pytest.raises(RuntimeError, match="out of memory"):
        cache.Reset(1, 2000, 16, 2, 64)
    assert cache.empty() and cache.n_pages() == 0 and cache.bytes() == 0
    with pytest.raises(mlb.MlbError, match="paged KV cache is empty"):
        cache.ReadDevice(0, None, None, None, 1)
