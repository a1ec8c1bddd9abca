"""Refusals of the paged attention's entry points that need no GPU: the checks come
before any device call."""
import ctypes

import pytest

import mini_llama_b200 as mlb
from mini_llama_b200 import _lib


def err(rc, text, code=-1):
    assert rc == code, (rc, _lib.lib().mlb_last_error())
    assert text.encode() in _lib.lib().mlb_last_error(), _lib.lib().mlb_last_error()


def test_wait_selftest_refuses_bad_arguments():
    f = _lib.lib().mlb_paged_attention_wait_selftest
    a, b, c = (ctypes.byref(ctypes.c_int()) for _ in range(3))
    err(f(0, 0, 1.0, None, b, c), "null output")
    err(f(0, 0, 1.0, a, b, None), "null output")
    err(f(0, 2, 1.0, a, b, c), "unknown activation type 2")
    for limit in (0.0, -1.0, 1001.0, float("nan")):
        with pytest.raises(mlb.MlbError, match="limit_ms"):
            mlb.paged_attention_wait_selftest(limit_ms=limit)
