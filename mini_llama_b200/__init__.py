"""mini_llama_b200 — B200 (sm_100a) decode forward path of mini-llama.

Python mirror of the reference's device-branch interface, over the C ABI of
include/mlb200.h (libmlb200.so). Names follow the reference
(include/mini_llama/cuda_quant.h, cuda_matmul.h, cuda_ops.h, cuda_attention.h,
cuda_kv_cache.h, forward.h); device memory is held in torch CUDA tensors,
which here are plumbing only -- every computation runs in this package's own
kernels. Errors raise ``MlbError`` (the reference's std::runtime_error) or
``MlbRangeError`` (std::out_of_range) with the reference's messages.
"""
from __future__ import annotations

import ctypes
import functools
import os

import numpy as np

from . import configs
from ._lib import MlbConfig, MlbError, MlbRangeError, check, lib, synth_lib
from .configs import (F32, Q4_0, Q4_1, Q8_0, W_BK, W_BQ, W_BV, W_DOWN, W_FFN_NORM,
                      W_FINAL_NORM, W_GATE, W_LM_HEAD, W_TOKEN_EMBEDDING, W_UP, W_WK, W_WO,
                      W_WQ, W_WV, W_ATTENTION_NORM)

ROPE_NORMAL, ROPE_NEOX = 0, 1
ROPE_NONE = -1  # MLB_ROPE_NONE: CudaPagedKvCache.AppendDevice stores rows as they are
ATTN_CPU_COMPAT, ATTN_STANDARD = 0, 1
KV_F32, KV_BF16 = 0, 1  # MLB_KV_F32, MLB_KV_BF16: KV cache element type of a Batch
ERR_TIMEOUT = -5  # MLB_ERR_TIMEOUT: a bounded device wait gave up

__all__ = [
    "F32", "Q8_0", "Q4_0", "Q4_1", "ROPE_NORMAL", "ROPE_NEOX", "ROPE_NONE", "ATTN_CPU_COMPAT",
    "ATTN_STANDARD", "Sampler", "MlbError", "MlbRangeError", "CudaQuantBuilt", "CudaDeviceCount",
    "CudaQ80LinearDeviceInput", "CudaQ40LinearDeviceInput", "CudaQ41LinearDeviceInput",
    "CudaLinearDeviceInput", "CudaQ80Linear", "CudaQ40Linear", "CudaQ41Linear", "CudaLinear",
    "CudaRmsNormDeviceWeight", "CudaSiluDeviceInput", "CudaElementwiseMulDeviceInput",
    "CudaElementwiseAddDeviceInput", "CudaSoftmax", "CudaEmbeddingLookupDeviceWeight",
    "CudaRopeDeviceInput", "CudaArgMax", "CudaLogProbs", "CudaKvCache",
    "CudaAttentionDecodeDeviceInput", "CudaPagedKvCache", "CudaPagedAttentionDeviceInput",
    "paged_attention_status", "paged_attention_wait_selftest",
    "QMatrix", "CudaModel", "Context", "Batch", "ForwardToken", "configs", "tp_plan", "nccl_unique_id",
]


_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch  # device memory and streams only

        _torch_module = torch
    return _torch_module


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    torch = _torch()
    if stream is None:
        return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    return ctypes.c_void_p(stream)


def CudaQuantBuilt() -> bool:
    """CudaQuantBuilt (include/mini_llama/cuda_quant.h:10)."""
    return bool(lib().mlb_built())


def CudaDeviceCount() -> int:
    """CudaDeviceCount (include/mini_llama/cuda_runtime.h:27)."""
    n = ctypes.c_int(0)
    check(lib().mlb_device_count(ctypes.byref(n)))
    return n.value


# ------------------------------------------------------------------ linear

def wait_selftest(which: int, limit_ms: float = 1.0, device_id: int = 0):
    """Runs one of the step kernel's bounded waits against something that
    never arrives (0: a ring slot's mbarrier, 1: a grid barrier) and returns
    the (status code, site) it recorded: (MLB_ERR_TIMEOUT, 900 + which) when
    the wait gave up after limit_ms."""
    code, where = ctypes.c_int(0), ctypes.c_int(0)
    check(lib().mlb_wait_selftest(device_id, which, float(limit_ms), ctypes.byref(code),
                                  ctypes.byref(where)))
    return code.value, where.value


def _linear_device_input(qtype, x, w_dev, block_count, weight_shape, device_id, stream=None):
    torch = _torch()
    if len(weight_shape) != 2:
        raise MlbError(-1, "expected weight shape [out_features, in_features]")
    out_f, in_f = int(weight_shape[0]), int(weight_shape[1])
    if x.dim() not in (1, 2):
        raise MlbError(-1, "expected x shape [in_features] or [batch, in_features]")
    if x.shape[-1] != in_f:
        raise MlbError(-1, f"dimension mismatch x={list(x.shape)} weight=[{out_f}, {in_f}]")
    rows = 1 if x.dim() == 1 else x.shape[0]
    x = x.contiguous()
    y = torch.empty((out_f,) if x.dim() == 1 else (rows, out_f), dtype=torch.float32,
                    device=x.device)
    check(lib().mlb_linear(qtype, _ptr(x), rows, in_f, _ptr(w_dev), block_count, out_f, _ptr(y),
                           device_id, _stream(stream)))
    return y


def CudaQ80LinearDeviceInput(x, w_dev, block_count, weight_shape, device_id=0, stream=None):
    """CudaQ80LinearDeviceInput (include/mini_llama/cuda_quant.h:18)."""
    return _linear_device_input(Q8_0, x, w_dev, block_count, weight_shape, device_id, stream)


def CudaQ40LinearDeviceInput(x, w_dev, block_count, weight_shape, device_id=0, stream=None):
    """CudaQ40LinearDeviceInput (include/mini_llama/cuda_quant.h:24)."""
    return _linear_device_input(Q4_0, x, w_dev, block_count, weight_shape, device_id, stream)


def CudaQ41LinearDeviceInput(x, w_dev, block_count, weight_shape, device_id=0, stream=None):
    """CudaQ41LinearDeviceInput (include/mini_llama/cuda_quant.h:30), with the CPU
    path's d*q + m dequantisation (src/quant.cc:455)."""
    return _linear_device_input(Q4_1, x, w_dev, block_count, weight_shape, device_id, stream)


def CudaLinearDeviceInput(x, w_dev, weight_shape, device_id=0, stream=None):
    """CudaLinearDeviceInput (include/mini_llama/cuda_matmul.h:18), F32 weights."""
    return _linear_device_input(F32, x, w_dev, int(weight_shape[0]) * int(weight_shape[1]),
                                weight_shape, device_id, stream)


def _linear_host(qtype, x, blocks, weight_shape, bias, device_id):
    x = np.ascontiguousarray(x, np.float32)
    blocks = np.ascontiguousarray(blocks)
    out_f, in_f = int(weight_shape[0]), int(weight_shape[1])
    rows = 1 if x.ndim == 1 else x.shape[0]
    nblk = out_f * in_f if qtype == F32 else out_f * ((in_f + 31) // 32)
    y = np.zeros((rows, out_f), np.float32)
    b = None if bias is None else np.ascontiguousarray(bias, np.float32)
    check(lib().mlb_linear_host(qtype, x.ctypes.data, rows, in_f, blocks.ctypes.data, nblk, out_f,
                                None if b is None else b.ctypes.data, y.ctypes.data, device_id))
    return y[0] if x.ndim == 1 else y


def CudaQ80Linear(x, blocks, weight_shape, bias=None, device_id=0):
    """CudaQ80Linear (include/mini_llama/cuda_quant.h:12): host in, host out."""
    return _linear_host(Q8_0, x, blocks, weight_shape, bias, device_id)


def CudaQ40Linear(x, blocks, weight_shape, bias=None, device_id=0):
    """CudaQ40Linear (include/mini_llama/cuda_quant.h:20)."""
    return _linear_host(Q4_0, x, blocks, weight_shape, bias, device_id)


def CudaQ41Linear(x, blocks, weight_shape, bias=None, device_id=0):
    """CudaQ41Linear (include/mini_llama/cuda_quant.h:26)."""
    return _linear_host(Q4_1, x, blocks, weight_shape, bias, device_id)


def CudaLinear(x, weight, bias=None, device_id=0):
    """CudaLinear (include/mini_llama/cuda_matmul.h:14): F32 weight [out, in]."""
    weight = np.ascontiguousarray(weight, np.float32)
    return _linear_host(F32, x, weight, weight.shape, bias, device_id)


# ------------------------------------------------------------- elementwise

def _empty_like(x):
    return _torch().empty_like(x)


def CudaRmsNormDeviceWeight(x, w, eps, device_id=0, stream=None):
    """CudaRmsNormDeviceWeight (include/mini_llama/cuda_ops.h:27)."""
    if x.dim() != 1 or w.dim() != 1:
        raise MlbError(-1, "RmsNorm: expected 1D tensors")
    if x.shape[0] != w.shape[0]:
        raise MlbError(-1, "RmsNorm: dimension mismatch")
    y = _empty_like(x)
    check(lib().mlb_rmsnorm(_ptr(x), _ptr(w), x.numel(), eps, _ptr(y), device_id, _stream(stream)))
    return y


def CudaSiluDeviceInput(x, device_id=0, stream=None):
    """CudaSiluDeviceInput (include/mini_llama/cuda_ops.h:29)."""
    y = _empty_like(x)
    check(lib().mlb_silu(_ptr(x), x.numel(), _ptr(y), device_id, _stream(stream)))
    return y


def CudaElementwiseMulDeviceInput(a, b, device_id=0, stream=None):
    """CudaElementwiseMulDeviceInput (include/mini_llama/cuda_ops.h:31)."""
    if a.shape != b.shape:
        raise MlbError(-1, f"ElementwiseMul: shape mismatch {list(a.shape)} vs {list(b.shape)}")
    y = _empty_like(a)
    check(lib().mlb_mul(_ptr(a), _ptr(b), a.numel(), _ptr(y), device_id, _stream(stream)))
    return y


def CudaElementwiseAddDeviceInput(a, b, device_id=0, stream=None):
    """CudaElementwiseAddDeviceInput (include/mini_llama/cuda_ops.h:33)."""
    if a.numel() != b.numel():
        raise MlbError(-1, f"ElementwiseAdd: shape mismatch {list(a.shape)} vs {list(b.shape)}")
    y = _empty_like(a)
    check(lib().mlb_add(_ptr(a), _ptr(b), a.numel(), _ptr(y), device_id, _stream(stream)))
    return y


def CudaSoftmax(x, device_id=0, stream=None):
    """CudaSoftmax (include/mini_llama/cuda_ops.h:19) on device data."""
    if x.dim() != 1:
        raise MlbError(-1, "Softmax: expected 1D tensor")
    y = _empty_like(x)
    check(lib().mlb_softmax(_ptr(x), x.numel(), _ptr(y), device_id, _stream(stream)))
    return y


def CudaEmbeddingLookupDeviceWeight(table, token_id, device_id=0, stream=None):
    """CudaEmbeddingLookupDeviceWeight (include/mini_llama/cuda_ops.h:23)."""
    vocab, dim = table.shape
    y = _torch().empty(dim, dtype=table.dtype, device=table.device)
    check(lib().mlb_embedding(_ptr(table), vocab, dim, int(token_id), _ptr(y), device_id,
                              _stream(stream)))
    return y


def CudaRopeDeviceInput(q, k, n_heads, n_kv_heads, head_dim, pos, theta,
                        rope_type=ROPE_NORMAL, device_id=0, stream=None):
    """CudaRopeDeviceInput (include/mini_llama/cuda_ops.h:37): in place."""
    check(lib().mlb_rope(_ptr(q), _ptr(k), n_heads, n_kv_heads, head_dim, pos, theta, rope_type,
                         device_id, _stream(stream)))


def CudaArgMax(x, device_id=0, stream=None) -> int:
    """ArgMax (src/ops.cc:220) on device logits; lowest index wins ties."""
    out = ctypes.c_int(0)
    check(lib().mlb_argmax(_ptr(x), x.numel(), ctypes.byref(out), device_id, _stream(stream)))
    return out.value


def _on_stream(call, device, stream):
    """Runs a call with `stream` (a cudaStream_t address) current on `device`, so
    that memory it allocates and frees is reused in that stream's order only."""
    torch = _torch()
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device)):
        return call()


def _raw_stream(index):
    """torch's current stream on a device, without the 2 us of a Stream object."""
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(index) if raw else torch.cuda.current_stream(index).cuda_stream


def _act_type(who, t):
    torch = _torch()
    if t.dtype is torch.float32:
        return 0  # MLB_ACT_F32
    if t.dtype is torch.bfloat16:
        return 1  # MLB_ACT_BF16
    raise MlbError(-1, f"{who}: expected float32 or bfloat16, got {t.dtype}")


def _on_device(who, name, t, index):
    if t.get_device() != index:
        raise MlbError(-1, f"{who}: {name} is on {t.device}, expected cuda:{index}")


def _int_tensor(who, name, t, shape, index):
    if t.dtype is not _torch().int32 or t.shape != shape or not t.is_contiguous():
        raise MlbError(-1, f"{who}: expected contiguous int32 {name} of shape {list(shape)}, got "
                           f"{t.dtype} {list(t.shape)}")
    if t.get_device() != index:
        raise MlbError(-1, f"{who}: {name} is on {t.device}, expected cuda:{index}")


def CudaLogProbs(logits, tokens, top_k=0, stream=None):
    """Log probability of tokens[row], entropy (nats) and the top_k (0..32) most
    likely tokens of every row of logits [rows, vocab] (fp32 or bf16; any row
    stride), lower index first among equals (mlb_logprobs). Returns (logprobs
    [rows], entropy [rows], top_ids int32 [rows, top_k], top_logprobs [rows,
    top_k]). A token outside [0, vocab) marks a padded row: its log probability
    is NaN. Runs on logits' device."""
    torch = _torch()
    who = "LogProbs"
    if logits.dim() == 1:
        logits = logits[None]
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise MlbError(-1, f"{who}: expected logits [rows, vocab], got {list(logits.shape)}")
    act = _act_type(who, logits)
    rows, vocab = logits.shape
    if not 0 <= top_k <= min(32, vocab):
        raise MlbError(-1, f"{who}: top_k must be 0 to {min(32, vocab)}, got {top_k}")
    if not logits.is_cuda:
        raise MlbError(-1, f"{who}: logits must be on a CUDA device")
    index = logits.get_device()
    _int_tensor(who, "tokens", tokens, (rows,), index)
    if stream is not None:
        return _on_stream(lambda: CudaLogProbs(logits, tokens, top_k), logits.device, stream)
    stride = logits.stride(0) if rows > 1 else vocab
    if logits.stride(1) != 1 or stride < vocab:
        logits, stride = logits.contiguous(), vocab
    # made like tensors at hand: torch.empty with a shape, a type and a device takes
    # twice the time, and a row's call is bound by its time on the host
    logprob = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    ids = tokens.new_empty(rows, top_k)
    top = logprob.new_empty(rows, top_k)
    check(lib().mlb_logprobs(act, logits.data_ptr(), stride, rows, vocab, tokens.data_ptr(), top_k,
                             logprob.data_ptr(), entropy.data_ptr(), ids.data_ptr(),
                             top.data_ptr(), index, _raw_stream(index)))
    return logprob, entropy, ids, top


# -------------------------------------------------------- KV cache, attention

class CudaKvCache:
    """CudaKvCache (include/mini_llama/cuda_kv_cache.h:9-57): fp32 keys and values
    [n_layers, max_seq_len, n_kv_heads, head_dim] on one device."""

    def __init__(self, n_layers=0, max_seq_len=0, n_kv_heads=0, head_dim=0, device_id=0):
        self.keys = self.values = None
        self._shape = (0, 0, 0, 0)
        self.device_id = device_id
        if n_layers:
            self.Reset(n_layers, max_seq_len, n_kv_heads, head_dim, device_id)

    def Reset(self, n_layers, max_seq_len, n_kv_heads, head_dim, device_id=0):
        torch = _torch()
        for name, v in (("n_layers", n_layers), ("max_seq_len", max_seq_len),
                        ("n_kv_heads", n_kv_heads), ("head_dim", head_dim)):
            if v <= 0:
                raise MlbError(-1, f"CudaKvCache: {name} must be positive")
        self.device_id = device_id
        self._shape = (n_layers, max_seq_len, n_kv_heads, head_dim)
        dev = torch.device("cuda", device_id)
        self.keys = torch.zeros(self._shape, dtype=torch.float32, device=dev)
        self.values = torch.zeros(self._shape, dtype=torch.float32, device=dev)

    def Clear(self):
        if self.keys is not None:
            self.keys.zero_()
            self.values.zero_()

    def empty(self):
        return self.keys is None

    def n_layers(self):
        return self._shape[0]

    def max_seq_len(self):
        return self._shape[1]

    def n_kv_heads(self):
        return self._shape[2]

    def head_dim(self):
        return self._shape[3]

    def bytes(self):
        return 0 if self.keys is None else self.keys.numel() * 4

    def WriteDevice(self, layer, pos, k, v, stream=None):
        L, S, KV, D = self._shape
        check(lib().mlb_kv_write(_ptr(self.keys) if self.keys is not None else None,
                                 _ptr(self.values) if self.values is not None else None,
                                 L, S, KV, D, layer, pos, _ptr(k.contiguous()),
                                 _ptr(v.contiguous()), self.device_id, _stream(stream)))

    def ReadKeyHead(self, layer, pos, kv_head):
        return self.keys[layer, pos, kv_head].cpu().numpy()

    def ReadValueHead(self, layer, pos, kv_head):
        return self.values[layer, pos, kv_head].cpu().numpy()


def CudaAttentionDecodeDeviceInput(q, kv_cache: CudaKvCache, layer, pos, n_heads, n_kv_heads,
                                   head_dim, device_id=0, mode=ATTN_STANDARD, stream=None):
    """CudaAttentionDecodeDeviceInput (include/mini_llama/cuda_attention.h:13).
    mode ATTN_STANDARD matches the reference GPU kernel; ATTN_CPU_COMPAT the CPU path."""
    torch = _torch()
    if q.numel() != n_heads * head_dim:
        raise MlbError(-1, "CudaAttentionDecodeDeviceInput: q shape mismatch")
    if kv_cache.empty():
        raise MlbError(-1, "CudaAttentionDecodeDeviceInput: CUDA KV cache is empty")
    if kv_cache.n_kv_heads() != n_kv_heads or kv_cache.head_dim() != head_dim:
        raise MlbError(-1, "CudaAttentionDecodeDeviceInput: KV cache shape or device does not "
                           "match attention shape")
    out = torch.empty(n_heads * head_dim, dtype=torch.float32, device=q.device)
    L, S, _, _ = kv_cache._shape
    check(lib().mlb_attention_decode(_ptr(q.contiguous()), _ptr(kv_cache.keys),
                                     _ptr(kv_cache.values), L, S, layer, pos, n_heads, n_kv_heads,
                                     head_dim, mode, _ptr(out), device_id, _stream(stream)))
    return out


def _row_stride(t):
    """Row stride of [rows, heads, head_dim] whose rows the kernels can read as
    they are (contiguous, 16-byte aligned), or 0."""
    rows, heads, dim = t.shape
    row = heads * dim
    if t.is_contiguous():
        stride = row
    else:
        stride, head, one = t.stride()
        if (one != 1 and dim > 1) or (head != dim and heads > 1):
            return 0
        if rows <= 1:
            stride = row
        elif stride < row:
            return 0
    return 0 if stride * t.element_size() % 16 or t.data_ptr() % 16 else stride


def _aligned_rows(t):
    stride = _row_stride(t)
    if stride == 0:
        t = t.clone(memory_format=_torch().contiguous_format)
        stride = t.shape[1] * t.shape[2]
    return t, stride


@functools.lru_cache(maxsize=4096)
def _paged_workspace(act, rows, n_seqs, n_heads, n_kv_heads, head_dim, page_size, max_pages,
                     device_id):
    n = ctypes.c_size_t()
    check(lib().mlb_paged_attention_workspace(act, rows, n_seqs, n_heads, n_kv_heads, head_dim,
                                              page_size, max_pages, device_id, ctypes.byref(n)))
    return n.value


class CudaPagedKvCache:
    """Keys and values of many sequences in a pool of n_pages pages of page_size
    tokens per layer (a multiple of 16), held as Q4_0 blocks: 4.5 bits per
    element (mlb_paged_kv_*). Which pages a sequence owns is the caller's, given
    to every call as device int32 tensors: row_offsets [n_seqs + 1] (which rows
    of the call belong to which sequence), seq_lens [n_seqs] (lengths with these
    rows, which are a sequence's last) and page_table [n_seqs, max_pages]. Rows
    behind the last sequence are left as they were; positions past the table or
    on a page outside the pool are neither stored nor seen. Calls do not
    synchronise and may be captured in a CUDA graph. head_dim: a multiple of 8
    up to 128."""

    def __init__(self, n_layers=0, n_pages=0, page_size=0, n_kv_heads=0, head_dim=0, device_id=0):
        self.pages = None
        self._shape = (0, 0, 0, 0, 0)
        self.device_id = device_id
        if n_layers:
            self.Reset(n_layers, n_pages, page_size, n_kv_heads, head_dim, device_id)

    def Reset(self, n_layers, n_pages, page_size, n_kv_heads, head_dim, device_id=0):
        torch = _torch()
        for name, v in (("n_layers", n_layers), ("n_pages", n_pages)):
            if v <= 0:
                raise MlbError(-1, f"CudaPagedKvCache: {name} must be positive")
        n = ctypes.c_size_t()
        check(lib().mlb_paged_kv_page_bytes(page_size, n_kv_heads, head_dim, ctypes.byref(n)))
        # empty until there is a pool of the new shape: the old one makes room for it
        self.pages, self._shape = None, (0, 0, 0, 0, 0)
        self.device_id = device_id
        self.pages = torch.zeros((n_layers, n_pages, n.value), dtype=torch.uint8,
                                 device=torch.device("cuda", device_id))
        self._shape = (n_layers, n_pages, page_size, n_kv_heads, head_dim)

    def Clear(self):
        if self.pages is not None:
            self.pages.zero_()

    def empty(self):
        return self.pages is None

    def n_layers(self):
        return self._shape[0]

    def n_pages(self):
        return self._shape[1]

    def page_size(self):
        return self._shape[2]

    def n_kv_heads(self):
        return self._shape[3]

    def head_dim(self):
        return self._shape[4]

    def bytes(self):
        return 0 if self.pages is None else self.pages.numel()

    def _layer(self, who, layer):
        if self.pages is None:
            raise MlbError(-1, f"{who}: paged KV cache is empty")
        if not 0 <= layer < self._shape[0]:
            raise MlbRangeError(f"{who}: layer out of range")

    def _sequences(self, who, row_offsets, seq_lens, page_table):
        """(n_seqs, max_pages) of a call's sequences."""
        n = seq_lens.numel()
        if page_table.dim() != 2 or page_table.shape[1] == 0:
            raise MlbError(-1, f"{who}: expected page_table [n_seqs, max_pages]")
        width = page_table.shape[1]
        _int_tensor(who, "seq_lens", seq_lens, (n,), self.device_id)
        _int_tensor(who, "row_offsets", row_offsets, (n + 1,), self.device_id)
        _int_tensor(who, "page_table", page_table, (n, width), self.device_id)
        return n, width

    def AppendDevice(self, layer, k, v, row_offsets, seq_lens, page_table, theta=10000.0,
                     rope_type=ROPE_NORMAL, q=None, q_out=None, stream=None):
        """Stores k and v [rows, n_kv_heads, head_dim] (fp32 or bf16) at their
        positions, k rotated on the way, and returns q [rows, n_heads, head_dim]
        rotated to the same positions, in q_out if given (q itself: in place;
        otherwise no part of q, k or v).
        rope_type ROPE_NONE stores k and returns q as they are."""
        who = "CudaPagedKvCache"
        self._layer(who, layer)
        n_layers, n_pages, page_size, kv, dim = self._shape
        if k.dim() != 3 or k.shape[1:] != (kv, dim) or v.shape != k.shape:
            raise MlbError(-1, f"{who}: expected k and v [rows, {kv}, {dim}], got "
                               f"{list(k.shape)} and {list(v.shape)}")
        act = _act_type(who, k)
        if v.dtype is not k.dtype:
            raise MlbError(-1, f"{who}: k and v differ in type")
        rows = k.shape[0]
        _on_device(who, "k", k, self.device_id)
        _on_device(who, "v", v, self.device_id)
        n_seqs, max_pages = self._sequences(who, row_offsets, seq_lens, page_table)
        if stream is not None:
            return _on_stream(lambda: self.AppendDevice(
                layer, k, v, row_offsets, seq_lens, page_table, theta, rope_type, q, q_out),
                self.pages.device, stream)
        k, ks = _aligned_rows(k)
        v, vs = _aligned_rows(v)
        heads = qs = qos = 0
        q_at = out_at = None
        if q is not None:
            if (q.dim() != 3 or q.shape[0] != rows or q.shape[2] != dim or q.shape[1] == 0
                    or q.dtype is not k.dtype):
                raise MlbError(-1, f"{who}: expected q [{rows}, n_heads, {dim}] of k's type, got "
                                   f"{q.dtype} {list(q.shape)}")
            _on_device(who, "q", q, self.device_id)
            heads = q.shape[1]
            if q_out is None:
                q_out = q.new_empty(rows, heads, dim)
                qos = heads * dim
            else:
                _on_device(who, "q_out", q_out, self.device_id)
                if q_out.shape == q.shape and q_out.dtype is q.dtype:
                    qos = _row_stride(q_out)
                if qos == 0:
                    raise MlbError(-1, f"{who}: q_out must be shaped like q, with 16-byte aligned "
                                       "rows")
            q, qs = _aligned_rows(q)
            q_at, out_at = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise MlbError(-1, f"{who}: q_out without q")
        check(lib().mlb_paged_kv_append(
            self.pages.data_ptr(), n_layers, n_pages, page_size, kv, dim, layer, act, k.data_ptr(),
            ks, v.data_ptr(), vs, q_at, qs, heads, out_at, qos, rows, n_seqs,
            row_offsets.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(), max_pages, theta,
            rope_type, self.device_id, _raw_stream(self.device_id)))
        return q_out

    def ReadDevice(self, layer, row_offsets, seq_lens, page_table, n_rows, stream=None):
        """fp32 keys and values [n_rows, n_kv_heads, head_dim] that the codes of
        the sequences' last rows stand for (row_offsets as in AppendDevice; whole
        sequences: the running sum of seq_lens). Rows that are not stored are 0."""
        torch = _torch()
        who = "CudaPagedKvCache"
        self._layer(who, layer)
        if n_rows < 0:
            raise MlbError(-1, f"{who}: negative row count")
        n_seqs, max_pages = self._sequences(who, row_offsets, seq_lens, page_table)
        if stream is not None:
            return _on_stream(lambda: self.ReadDevice(layer, row_offsets, seq_lens, page_table,
                                                      n_rows), self.pages.device, stream)
        n_layers, n_pages, page_size, kv, dim = self._shape
        k = self.pages.new_empty(n_rows, kv, dim, dtype=torch.float32)
        v = torch.empty_like(k)
        check(lib().mlb_paged_kv_read(
            self.pages.data_ptr(), n_layers, n_pages, page_size, kv, dim, layer, n_rows, n_seqs,
            row_offsets.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(), max_pages,
            k.data_ptr(), v.data_ptr(), self.device_id, _raw_stream(self.device_id)))
        return k, v


def paged_attention_status(device_id=0):
    """(status code, site) of the last bounded wait that gave up in the prompt
    form of CudaPagedAttentionDeviceInput since the last call, (0, 0) if none
    did (mlb_paged_attention_status); rows without a result are NaN. Waits for
    the device."""
    code, where = ctypes.c_int(0), ctypes.c_int(0)
    check(lib().mlb_paged_attention_status(device_id, ctypes.byref(code), ctypes.byref(where)))
    return code.value, where.value


def paged_attention_wait_selftest(bf16=False, limit_ms: float = 1.0, device_id: int = 0):
    """Runs the prompt form on 8 rows with a barrier that never completes and returns
    (status code, site, rows that became NaN): (MLB_ERR_TIMEOUT, 1001 .. 1011, 8) when
    its waits gave up after limit_ms (mlb_paged_attention_wait_selftest)."""
    code, where, rows = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
    check(lib().mlb_paged_attention_wait_selftest(device_id, int(bool(bf16)), float(limit_ms),
                                                  ctypes.byref(code), ctypes.byref(where),
                                                  ctypes.byref(rows)))
    return code.value, where.value, rows.value


def CudaPagedAttentionDeviceInput(q, kv_cache: CudaPagedKvCache, layer, row_offsets, seq_lens,
                                  page_table, n_heads, n_kv_heads, head_dim, scale=None, out=None,
                                  stream=None):
    """Attention of q [rows, n_heads, head_dim] (fp32 or bf16), each row over the
    positions of its sequence up to its own (mlb_paged_attention): one row per
    sequence while decoding, a few to check drafted tokens, many for a prompt
    (long decoding sequences in a call of their own: beside a prompt they are slow).
    scale defaults to 1 / sqrt(head_dim). A row that sees nothing gets zeros. Rows of
    out must not overlap rows of q (side by side in one buffer they do not)."""
    who = "CudaPagedAttention"
    kv_cache._layer(who, layer)
    n_layers, n_pages, page_size, kv, dim = kv_cache._shape
    if kv != n_kv_heads or dim != head_dim:
        raise MlbError(-1, f"{who}: KV cache shape does not match attention shape")
    if n_heads <= 0 or n_heads % n_kv_heads != 0:
        raise MlbError(-1, f"{who}: n_heads must be divisible by n_kv_heads")
    if q.dim() != 3 or q.shape[1:] != (n_heads, head_dim):
        raise MlbError(-1, f"{who}: expected q [rows, {n_heads}, {head_dim}], got {list(q.shape)}")
    act = _act_type(who, q)
    index = kv_cache.device_id
    _on_device(who, "q", q, index)
    n_seqs, max_pages = kv_cache._sequences(who, row_offsets, seq_lens, page_table)
    if stream is not None:
        return _on_stream(lambda: CudaPagedAttentionDeviceInput(
            q, kv_cache, layer, row_offsets, seq_lens, page_table, n_heads, n_kv_heads, head_dim,
            scale, out), q.device, stream)
    rows = q.shape[0]
    if out is None:
        out = q.new_empty(rows, n_heads, head_dim)
        out_stride = n_heads * head_dim
    else:
        _on_device(who, "out", out, index)
        out_stride = _row_stride(out) if out.shape == q.shape and out.dtype is q.dtype else 0
        if out_stride == 0:
            raise MlbError(-1, f"{who}: out must be shaped like q, with 16-byte aligned rows")
    q, q_stride = _aligned_rows(q)
    size = _paged_workspace(act, rows, n_seqs, n_heads, n_kv_heads, head_dim, page_size,
                            max_pages, index)
    ws = kv_cache.pages.new_empty(size) if size else None
    check(lib().mlb_paged_attention(
        kv_cache.pages.data_ptr(), n_layers, n_pages, page_size, kv, dim, layer, act, q.data_ptr(),
        q_stride, n_heads, rows, n_seqs, row_offsets.data_ptr(), seq_lens.data_ptr(),
        page_table.data_ptr(), max_pages, head_dim ** -0.5 if scale is None else scale,
        out.data_ptr(), out_stride, ws.data_ptr() if size else None, size, index,
        _raw_stream(index)))
    return out


# ------------------------------------------------------ prepared weight GEMV

class QMatrix:
    """A weight repacked into the B200 GEMV layout (the decode path's format)."""

    def __init__(self, handle, qtype, out_features, in_features, device_id=0):
        self.h = handle
        self.qtype, self.out_features, self.in_features = qtype, out_features, in_features
        self.device_id = device_id

    @classmethod
    def from_gguf(cls, qtype, blocks, out_features, in_features, device_id=0):
        """blocks: host numpy uint8/float32 array, or a CUDA tensor, in GGUF layout."""
        h = ctypes.c_void_p()
        if isinstance(blocks, np.ndarray):
            blocks = np.ascontiguousarray(blocks)
            check(lib().mlb_qmatrix_create(qtype, blocks.ctypes.data, 1, out_features, in_features,
                                           device_id, ctypes.byref(h)))
        else:
            check(lib().mlb_qmatrix_create(qtype, _ptr(blocks), 0, out_features, in_features,
                                           device_id, ctypes.byref(h)))
        return cls(h, qtype, out_features, in_features, device_id)

    @classmethod
    def synthesize(cls, qtype, out_features, in_features, seed, stream_id=0, raw=False,
                   device_id=0):
        h = ctypes.c_void_p()
        check(lib().mlb_qmatrix_synthesize(qtype, out_features, in_features, seed, stream_id,
                                           int(raw), device_id, ctypes.byref(h)))
        return cls(h, qtype, out_features, in_features, device_id)

    def gemv(self, x, y=None, stream=None):
        torch = _torch()
        rows = 1 if x.dim() == 1 else x.shape[0]
        if y is None:
            y = torch.empty((rows, self.out_features) if x.dim() == 2 else (self.out_features,),
                            dtype=torch.float32, device=x.device)
        check(lib().mlb_qmatrix_gemv(self.h, _ptr(x), rows, _ptr(y), _stream(stream)))
        return y

    def gemm(self, x, y=None, stream=None):
        """y = W x on the tensor cores (mlb_qmatrix_gemm), any row count."""
        torch = _torch()
        rows = 1 if x.dim() == 1 else x.shape[0]
        if y is None:
            y = torch.empty((rows, self.out_features) if x.dim() == 2 else (self.out_features,),
                            dtype=torch.float32, device=x.device)
        check(lib().mlb_qmatrix_gemm(self.h, _ptr(x), rows, _ptr(y), _stream(stream)))
        return y

    def dequant(self, out=None, stream=None):
        """fp32 [out_features, in_features] on the device, decoded from the
        repacked layout (DequantizeFromQ80/Q40/Q41, src/quant.cc:170-361)."""
        torch = _torch()
        if out is None:
            out = torch.empty((self.out_features, self.in_features), dtype=torch.float32,
                              device=f"cuda:{self.device_id}")
        check(lib().mlb_qmatrix_dequant(self.h, _ptr(out), _stream(stream)))
        return out

    def gguf_bytes(self):
        return lib().mlb_qmatrix_bytes(self.h)

    def __del__(self):
        try:
            if self.h:
                lib().mlb_qmatrix_destroy(self.h)
                self.h = None
        except Exception:
            pass


# ------------------------------------------------------------ model, context

class CudaModel:
    """Device-resident model: UploadModelWeightsToCuda (src/model.cc:345-374) as
    set_weight/finalize, or seeded on-device synthesis. tp_size > 1 keeps this
    rank's tensor-parallel shard (nccl_id: 128 bytes from nccl_unique_id())."""

    def __init__(self, cfg: dict, device_id=0, tp_rank=0, tp_size=1, nccl_id: bytes | None = None):
        self.cfg = dict(cfg)
        self.device_id = device_id
        c = MlbConfig(**{k: cfg[k] for k, _ in MlbConfig._fields_})
        h = ctypes.c_void_p()
        idbuf = None if nccl_id is None else ctypes.create_string_buffer(bytes(nccl_id), 128)
        check(lib().mlb_model_create(ctypes.byref(c), device_id, tp_rank, tp_size, idbuf,
                                     ctypes.byref(h)))
        self.h = h

    @classmethod
    def from_gguf(cls, path: str, device_id=0, tp_rank=0, tp_size=1, nccl_id: bytes | None = None,
                  max_seq_len: int = 0):
        """LoadGgufModel + UploadModelWeightsToCuda (mlb_model_load_gguf): the model
        of a GGUF v3 file, uploaded from the mapped file and finalized.
        max_seq_len > 0 replaces the file's context_length. The bytes copied to
        the device are in .gguf_bytes."""
        self = cls.__new__(cls)
        self.cfg = read_gguf_config(path)
        if max_seq_len > 0:
            self.cfg["max_seq_len"] = max_seq_len
        self.device_id = device_id
        h = ctypes.c_void_p()
        n = ctypes.c_size_t()
        idbuf = None if nccl_id is None else ctypes.create_string_buffer(bytes(nccl_id), 128)
        check(lib().mlb_model_load_gguf(os.fsencode(path), device_id, tp_rank, tp_size, idbuf,
                                        int(max_seq_len), ctypes.byref(h), ctypes.byref(n)))
        self.h = h
        self.gguf_bytes = n.value
        return self

    def set_weight(self, kind, layer, qtype, rows, cols, data: np.ndarray):
        data = np.ascontiguousarray(data)
        check(lib().mlb_model_set_weight(self.h, kind, layer, qtype, rows, cols, data.ctypes.data,
                                         data.nbytes))

    def load(self, weights):
        """weights: iterable of (kind, layer, qtype, rows, cols, array)."""
        for kind, layer, qtype, rows, cols, arr in weights:
            self.set_weight(kind, layer, qtype, rows, cols, arr)
        self.finalize()
        return self

    def synthesize(self, qtype, seed, with_bias=False):
        check(lib().mlb_model_synthesize(self.h, qtype, seed, int(with_bias)))
        return self

    def finalize(self):
        check(lib().mlb_model_finalize(self.h))
        return self

    def bytes(self):
        r, s = ctypes.c_size_t(), ctypes.c_size_t()
        check(lib().mlb_model_bytes(self.h, ctypes.byref(r), ctypes.byref(s)))
        return r.value, s.value

    def context(self, attention_mode=ATTN_CPU_COMPAT, step_kernel=None, kv_type=0):
        return Context(self, attention_mode, step_kernel, kv_type)

    def close(self):
        if getattr(self, "h", None):
            lib().mlb_model_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Context:
    """MiniLlamaContext with its CUDA KV cache (include/mini_llama/context.h)."""

    def __init__(self, model: CudaModel, attention_mode=ATTN_CPU_COMPAT, step_kernel=None,
                 kv_type: int = 0):
        """kv_type: KV_F32 (the reference's fp32 cache) or KV_BF16 (step kernel only)."""
        self.model = model
        h = ctypes.c_void_p()
        check(lib().mlb_context_create_kv(model.h, attention_mode, int(kv_type), ctypes.byref(h)))
        self.h = h
        self.pos = 0
        self.token_history = []
        if step_kernel is not None:
            self.set_step_kernel(step_kernel)

    def set_step_kernel(self, enable: bool):
        """True: one persistent kernel per decode step; False: one kernel per op."""
        check(lib().mlb_context_set_step_kernel(self.h, 1 if enable else 0))

    def step_kernel(self) -> bool:
        return bool(lib().mlb_context_step_kernel(self.h))

    def decode_sample(self, sampler: "Sampler", token: int, pos: int, n_steps: int,
                      temperature: float = 0.0, top_k: int = 0) -> list:
        """decode_greedy with the sampler's choice at every step (mlb_decode_sample)."""
        out = np.empty(max(n_steps, 1), np.int32)
        check(lib().mlb_decode_sample(self.h, sampler.h, float(temperature), int(top_k),
                                      int(token), int(pos), int(n_steps), out.ctypes.data))
        return [int(t) for t in out[:n_steps]]

    def step_trace(self, enable: bool):
        """Records per-phase times of later step-kernel steps (diagnostic)."""
        check(lib().mlb_context_step_trace(self.h, 1 if enable else 0))

    def step_trace_read(self) -> np.ndarray:
        """Global-timer stamps (ns) of the last traced step, [phase][cta][2]:
        start of each phase's work after its barrier, end before the next.
        Phases: per layer QKV, attention, wo, gate/up, w_down; then lm_head."""
        n, g = ctypes.c_int(0), ctypes.c_int(0)
        check(lib().mlb_context_step_trace_read(self.h, None, 0, ctypes.byref(n),
                                                ctypes.byref(g)))
        out = np.zeros((n.value, g.value, 2), np.uint64)
        check(lib().mlb_context_step_trace_read(self.h, out.ctypes.data, out.size,
                                                ctypes.byref(n), ctypes.byref(g)))
        return out

    def forward_token(self, token: int, pos: int) -> np.ndarray:
        """ForwardToken's device branch (src/forward.cc:776-794): host logits."""
        out = np.empty(self.model.cfg["vocab_size"], np.float32)
        check(lib().mlb_forward_token(self.h, int(token), int(pos), out.ctypes.data))
        return out

    def forward_token_device(self, token: int, pos: int) -> int:
        """Asynchronous step; returns the device address of the logits."""
        p = ctypes.c_void_p()
        check(lib().mlb_forward_token_device(self.h, int(token), int(pos), ctypes.byref(p)))
        return p.value

    def sync(self):
        check(lib().mlb_context_sync(self.h))

    def decode_greedy(self, token: int, pos: int, n_steps: int) -> list:
        out = np.empty(max(n_steps, 1), np.int32)
        check(lib().mlb_decode_greedy(self.h, int(token), int(pos), int(n_steps), out.ctypes.data))
        return [int(t) for t in out[:n_steps]]

    def reset(self):
        check(lib().mlb_context_reset(self.h))
        self.pos = 0
        self.token_history = []

    def fill_kv(self, n_pos: int, seed: int, scale: float = 1.25):
        """Seeded K/V rows for positions [0, n_pos) (mlb_context_fill_kv)."""
        check(lib().mlb_context_fill_kv(self.h, int(n_pos), int(seed), float(scale)))

    def forward_batch(self, tokens, positions) -> np.ndarray:
        """ForwardBatch (src/batch.cc:35-50): every token at its position, the
        last token's logits (mlb_forward_batch)."""
        t = np.ascontiguousarray(tokens, np.int32)
        p = np.ascontiguousarray(positions, np.int32)
        out = np.empty(self.model.cfg["vocab_size"], np.float32)
        check(lib().mlb_forward_batch(self.h, len(t), t.ctypes.data, p.ctypes.data,
                                      out.ctypes.data))
        return out

    def stream(self) -> int:
        return lib().mlb_context_stream(self.h) or 0

    def kernels_per_step(self) -> int:
        return lib().mlb_context_kernels_per_step(self.h)

    def close(self):
        if getattr(self, "h", None):
            lib().mlb_context_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Sampler:
    """MiniSampler (include/mini_llama/sampler.h) on the device: a std::mt19937
    seeded with `seed` (0: a random seed) whose state stays on device_id."""

    def __init__(self, seed: int = 0, device_id: int = 0):
        h = ctypes.c_void_p()
        check(lib().mlb_sampler_create(int(device_id), int(seed), ctypes.byref(h)))
        self.h = h
        self.device_id = device_id

    def sample(self, logits_ptr: int, n: int, temperature: float = 0.0, top_k: int = 0) -> int:
        """MiniSampler::Sample over n fp32 logits at device address logits_ptr."""
        out = ctypes.c_int(-1)
        check(lib().mlb_sample(self.h, ctypes.c_void_p(logits_ptr), int(n), float(temperature),
                               int(top_k), ctypes.byref(out)))
        return out.value

    def close(self):
        if getattr(self, "h", None):
            lib().mlb_sampler_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Batch:
    """n_seqs sequences decoded together (mlb_batch_*), each with its own KV cache."""

    def __init__(self, model: CudaModel, n_seqs: int, attention_mode=ATTN_CPU_COMPAT,
                 kv_type: int = 0):
        """kv_type: KV_F32 (the reference's fp32 cache) or KV_BF16."""
        self.model = model
        self.n_seqs = n_seqs
        self.kv_type = kv_type
        h = ctypes.c_void_p()
        check(lib().mlb_batch_create_kv(model.h, int(n_seqs), attention_mode, int(kv_type),
                                        ctypes.byref(h)))
        self.h = h

    def reset(self):
        check(lib().mlb_batch_reset(self.h))

    def fill_kv(self, seq: int, n_pos: int, seed: int, scale: float = 1.25):
        check(lib().mlb_batch_fill_kv(self.h, int(seq), int(n_pos), int(seed), float(scale)))

    def forward(self, seqs, tokens, positions, logits=False):
        """One pass of rows; returns (next greedy ids, logits [rows, vocab] or None)."""
        s = np.ascontiguousarray(seqs, np.int32)
        t = np.ascontiguousarray(tokens, np.int32)
        p = np.ascontiguousarray(positions, np.int32)
        nxt = np.empty(len(t), np.int32)
        lg = np.empty((len(t), self.model.cfg["vocab_size"]), np.float32) if logits else None
        check(lib().mlb_batch_forward(self.h, len(t), s.ctypes.data, t.ctypes.data, p.ctypes.data,
                                      lg.ctypes.data if logits else None, nxt.ctypes.data))
        return [int(v) for v in nxt], lg

    def decode_greedy(self, tokens, positions, n_steps: int) -> np.ndarray:
        """[n_steps, n_seqs] greedy ids, all sequences in lockstep."""
        t = np.ascontiguousarray(tokens, np.int32)
        p = np.ascontiguousarray(positions, np.int32)
        out = np.empty((max(n_steps, 1), self.n_seqs), np.int32)
        check(lib().mlb_batch_decode_greedy(self.h, t.ctypes.data, p.ctypes.data, int(n_steps),
                                            out.ctypes.data))
        return out[:n_steps]

    def stream(self) -> int:
        return lib().mlb_batch_stream(self.h) or 0

    def kernels_per_step(self) -> int:
        return lib().mlb_batch_kernels_per_step(self.h)

    def close(self):
        if getattr(self, "h", None):
            lib().mlb_batch_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def ForwardToken(ctx: Context, token: int) -> np.ndarray:
    """ForwardToken(ctx, model, token) (include/mini_llama/forward.h:11) at ctx.pos."""
    return ctx.forward_token(token, ctx.pos)


def read_gguf_config(path: str) -> dict:
    """The model config LoadGgufModel builds from a GGUF file (host only)."""
    c = MlbConfig()
    check(lib().mlb_gguf_read_config(os.fsencode(path), ctypes.byref(c)))
    return {k: getattr(c, k) for k, _ in MlbConfig._fields_}


def tp_plan(cfg: dict, tp_rank: int, tp_size: int) -> dict:
    """The tensor-parallel shard of one rank (host only; see mlb_tp_plan)."""
    from ._lib import MlbTpShard

    c = MlbConfig(**{k: cfg[k] for k, _ in MlbConfig._fields_})
    out = MlbTpShard()
    check(lib().mlb_tp_plan(ctypes.byref(c), int(tp_rank), int(tp_size), ctypes.byref(out)))
    return {k: getattr(out, k) for k, _ in MlbTpShard._fields_}


def nccl_unique_id() -> bytes:
    buf = ctypes.create_string_buffer(128)
    check(lib().mlb_nccl_unique_id(buf))
    return buf.raw
