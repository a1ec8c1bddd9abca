"""Argument checks of the paged-cache and log-probability entry points: every
bad argument is refused before any device call, so these run with no GPU."""
import ctypes

import pytest

import mini_llama_b200 as mlb
from mini_llama_b200 import _lib

P = ctypes.c_void_p(256)  # never dereferenced: the checks come first
ODD = ctypes.c_void_p(260)


def err(rc, text, code=-1):
    assert rc == code, (rc, _lib.lib().mlb_last_error())
    assert text.encode() in _lib.lib().mlb_last_error(), _lib.lib().mlb_last_error()


@pytest.mark.parametrize("page,kv,hd,want", [
    (16, 1, 32, 576), (16, 8, 128, 8 * 2304), (64, 8, 128, 4 * 8 * 2304), (48, 6, 48, 3 * 6 * 1152),
    (16, 2, 8, 2 * 576), (32, 1, 96, 2 * 1728)])
def test_page_bytes(page, kv, hd, want):
    n = ctypes.c_size_t()
    assert _lib.lib().mlb_paged_kv_page_bytes(page, kv, hd, ctypes.byref(n)) == 0
    assert n.value == want


def test_shapes_are_refused():
    f = _lib.lib().mlb_paged_kv_page_bytes
    n = ctypes.c_size_t()
    err(f(0, 1, 32, ctypes.byref(n)), "page_size must be a positive multiple of 16")
    err(f(24, 1, 32, ctypes.byref(n)), "page_size must be a positive multiple of 16")
    err(f(16, 0, 32, ctypes.byref(n)), "n_kv_heads must be positive")
    for hd in (0, 4, 36, 136):
        err(f(16, 1, hd, ctypes.byref(n)), "head_dim must be a multiple of 8 up to 128")
    err(f(16, 1, 32, None), "null output")


def append(**kw):
    a = dict(pages=P, layers=2, n_pages=4, page=16, kv=2, hd=64, layer=0, act=0, k=P, ks=128, v=P,
             vs=128, q=P, qs=256, heads=4, qo=P, qos=256, rows=3, seqs=1, offs=P, lens=P, table=P,
             width=2, theta=1e4, rope=0)
    a.update(kw)
    return _lib.lib().mlb_paged_kv_append(*a.values(), 0, None)


def test_append_is_refused():
    err(append(pages=None), "paged KV cache is empty")
    err(append(pages=ODD), "pages must be 16-byte aligned")
    err(append(layer=2), "layer out of range", -2)
    err(append(layer=-1), "layer out of range", -2)
    err(append(act=2), "unknown activation type 2")
    err(append(rope=3), "unknown rope type 3")
    err(append(theta=float("nan")), "theta must be finite and positive")
    err(append(theta=-1.0), "theta must be finite and positive")
    err(append(rows=-1), "negative row or sequence count")
    err(append(width=0), "at least one column")
    err(append(width=1 << 30), "more than 2e9 positions")
    err(append(offs=None), "null row_offsets")
    err(append(k=None), "null k")
    err(append(v=ODD), "rows of v must be 16-byte aligned")
    err(append(ks=100), "row stride of k is smaller than a row")
    err(append(vs=129), "rows of v must be 16-byte aligned")
    err(append(act=1, qs=260), "rows of q must be 16-byte aligned")
    err(append(qo=None), "null q_out")
    err(append(heads=-1), "negative head count")


def attend(**kw):
    a = dict(pages=P, layers=2, n_pages=4, page=16, kv=2, hd=64, layer=0, act=0, q=P, qs=256,
             heads=4, rows=3, seqs=1, offs=P, lens=P, table=P, width=2, scale=0.1, out=P, outs=256,
             ws=P, wsn=1 << 30)
    a.update(kw)
    return _lib.lib().mlb_paged_attention(*a.values(), 0, None)


def test_attention_is_refused():
    err(attend(heads=3), "divisible by n_kv_heads")
    err(attend(heads=0), "n_heads must be positive")
    err(attend(scale=float("inf")), "scale must be finite")
    err(attend(out=None), "null out")
    err(attend(out=P), "must not overlap")
    err(attend(qs=255), "row stride of q is smaller than a row")
    err(attend(table=None), "page_table")
    err(attend(layer=9), "layer out of range", -2)
    n = ctypes.c_size_t()
    f = _lib.lib().mlb_paged_attention_workspace
    err(f(0, 1, 1, 4, 2, 64, 16, 8, 0, None), "null output")
    err(f(5, 1, 1, 4, 2, 64, 16, 8, 0, ctypes.byref(n)), "unknown activation type")
    err(f(0, 1, 1, 4, 2, 64, 16, 0, 0, ctypes.byref(n)), "page_table")
    err(f(0, 1, 1, 4, 2, 64, 24, 8, 0, ctypes.byref(n)), "multiple of 16")
    err(f(0, -1, 1, 4, 2, 64, 16, 8, 0, ctypes.byref(n)), "negative row or sequence count")


def read(**kw):
    a = dict(pages=P, layers=2, n_pages=4, page=16, kv=2, hd=64, layer=0, rows=3, seqs=1, offs=P,
             lens=P, table=P, width=2, k=P, v=P)
    a.update(kw)
    return _lib.lib().mlb_paged_kv_read(*a.values(), 0, None)


def test_read_is_refused():
    err(read(k=None), "null k_out")
    err(read(v=ODD), "rows of v_out must be 16-byte aligned")
    err(read(n_pages=0), "paged KV cache is empty")


def logprobs(**kw):
    a = dict(act=0, x=P, stride=100, rows=2, vocab=100, tok=P, k=3, lp=P, ent=P, ids=P, top=P)
    a.update(kw)
    return _lib.lib().mlb_logprobs(*a.values(), 0, None)


def test_logprobs_are_refused():
    err(logprobs(act=7), "unknown activation type 7")
    err(logprobs(rows=-1), "negative row count")
    err(logprobs(vocab=0), "empty logits")
    err(logprobs(stride=99), "row stride is smaller than a row")
    err(logprobs(k=33), "top_k must be 0 to 32")
    err(logprobs(vocab=2, k=3), "top_k must be 0 to 2")
    err(logprobs(k=-1), "top_k must be 0 to 32")
    err(logprobs(tok=None), "null pointer")
    err(logprobs(ids=None), "null pointer")
    err(logprobs(x=ctypes.c_void_p(257)), "logits are unaligned")


def test_python_forms_refuse_before_the_device():
    torch = pytest.importorskip("torch")
    with pytest.raises(mlb.MlbError, match="n_pages must be positive"):
        mlb.CudaPagedKvCache(1, 0, 16, 2, 64)
    with pytest.raises(mlb.MlbError, match="multiple of 16"):
        mlb.CudaPagedKvCache(1, 4, 20, 2, 64)
    assert mlb.CudaPagedKvCache().empty() and mlb.CudaPagedKvCache().bytes() == 0
    with pytest.raises(mlb.MlbError, match="paged KV cache is empty"):
        mlb.CudaPagedKvCache().AppendDevice(0, None, None, None, None, None)
    with pytest.raises(mlb.MlbError, match="expected logits"):
        mlb.CudaLogProbs(torch.zeros(2, 3, 4), None)
