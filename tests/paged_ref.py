"""Plain 64-bit forms of the paged-cache operators for the tests."""
import ctypes
import math

import numpy as np
import torch

from mini_llama_b200 import _lib


def quantise(x):
    """fp32 [..., hd] -> float64 values of its Q4_0 blocks, with the host
    quantiser that the weight generator uses (block by block, partial last)."""
    lib = _lib.synth_lib()
    rows = np.ascontiguousarray(x.float().cpu().numpy()).reshape(-1, x.shape[-1])
    hd = rows.shape[1]
    out = np.empty(rows.shape, np.float64)
    buf = np.zeros(18, np.uint8)
    for r in range(rows.shape[0]):
        for b in range(0, hd, 32):
            n = min(32, hd - b)
            src = np.ascontiguousarray(rows[r, b:b + n])
            lib.mlbs_quantize_block(2, src.ctypes.data, n, buf.ctypes.data)
            d = np.float64(buf[:2].view(np.float16)[0])
            codes = np.concatenate([buf[2:] & 15, buf[2:] >> 4]).astype(np.float64) - 8.0
            out[r, b:b + n] = codes[:n] * d
    return torch.from_numpy(out.reshape(x.shape))


def rotate(x, pos, theta, neox):
    """float64 rotation of x [rows, heads, hd] by its rows' positions."""
    x = x.double().cpu()
    hd = x.shape[-1]
    j = torch.arange(hd // 2, dtype=torch.float64)
    a = torch.as_tensor(pos, dtype=torch.float64)[:, None] * theta ** (-2.0 * j / hd)
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    i0 = torch.arange(hd // 2) if neox else 2 * torch.arange(hd // 2)
    i1 = i0 + (hd // 2 if neox else 1)
    y = torch.empty_like(x)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def attention(q, k, v, length, n, scale, absent=()):
    """float64 attention of one sequence's last n rows q [n, H, hd] over k, v
    [length, KV, hd]; positions in `absent` are not there. Returns (out, sum of
    p|v|, (largest sum |q||k| scale, largest |v|)) -- for the error bounds."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    H, KV = q.shape[1], k.shape[1]
    k = k.repeat_interleave(H // KV, 1)
    v = v.repeat_interleave(H // KV, 1)
    s = torch.einsum("ihd,thd->hit", q, k) * scale
    big = torch.einsum("ihd,thd->hit", q.abs(), k.abs()) * abs(scale)
    pos = torch.arange(length - n, length)
    seen = torch.arange(length)[None] <= pos[:, None]
    for t in absent:
        seen[:, t] = False
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(seen.any(-1)[:, None], p, torch.zeros_like(p))  # rows that see nothing
    top = big.masked_fill(~seen, 0.0).amax(-1) if length else torch.zeros(H, n)
    return (torch.einsum("hit,thd->ihd", p, v), torch.einsum("hit,thd->ihd", p, v.abs()),
            (top.transpose(0, 1)[..., None], v.abs().amax((0, 2))[None, :, None]))


def prompt_form(rows, n_seqs, kv, group, dtype):
    """Whether a call takes the prompt form (mlb_paged_attention's rule)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    f32 = dtype == torch.float32
    units, each = n_seqs * kv, -(-rows * group // n_seqs)
    ctas = units * -(-each // (128 if f32 else 256))
    return (-(-ctas // sms) * (2.1 if f32 else 1.65)
            < units * -(-each // 16) * (2.05 if f32 else 1.5) / (3 * sms))


def attention_bound(out, vabs, top, length, dtype, prompt=False):
    """Largest error of the kernels. Scores: queries kept to 2^-22 and up to 16
    truncated adds of 2^-23 per product, so at most top * 2^-18 each, doubled by
    numerator and denominator; p: exp 2^-21, P dV kept to 2^-21 (bf16 calls: two
    fp16 roundings, 2^-10), sums over the length one truncated add per 16 tokens
    and warp. An fp16 below 2^-14 is off by up to 2^-25 instead: P dV is scaled by
    2^F, the smaller of 2^15 and what brings the largest dV to at least 2^13, so
    that is the larger of 2^-40 and 2^-38 of the largest dV for each token, times
    codes up to 8 (the largest |v| is at most 8 dV, and at least 6 of them): per
    token 2^-37 or 2^-35 / 6 of the largest |v|.

    The prompt form adds: K and V in fp16, 2^-11 of each (fp32 calls: pairs that
    hold them whole, three products, so 48 adds to a score and three per 16 tokens
    to a sum), P in fp16, 2^-11, lifted by 2^7 (bf16 calls: 2^3), so that what it
    loses below 2^-14 is 2^-32 (2^-28) of the largest |v| per token."""
    top, vmax = top
    floor = length * torch.clamp(vmax * 2.0 ** -35 / 6, min=2.0 ** -37)
    rel = top * 2.0 ** -17 + (16 + length / 32) * 2.0 ** -22
    if prompt:
        floor = floor + length * vmax * 2.0 ** (-28 if dtype == torch.bfloat16 else -32)
        rel = top * 2.0 ** -16 + (16 + length / 8) * 2.0 ** -22
        if dtype == torch.bfloat16:
            rel = rel + (2 * top + 2) * 2.0 ** -11
    if dtype == torch.bfloat16:
        return vabs * (rel + 2.0 ** -10) + floor + out.abs() * 2.0 ** -8
    return vabs * rel + floor + out.abs() * 2.0 ** -24


class Seqs:
    """Ragged sequences over a shuffled pool."""

    def __init__(self, new, lens, page, extra=2, seed=0, device="cuda"):
        self.new, self.lens, self.page = list(new), list(lens), page
        g = torch.Generator().manual_seed(seed)
        counts = [(n + page - 1) // page for n in lens]
        self.n_pages = sum(counts) + extra
        ids = torch.randperm(self.n_pages, generator=g).tolist()
        self.ids, at = [], 0
        for c in counts:
            self.ids.append(ids[at:at + c])
            at += c
        self.spare = ids[at:]
        width = max(1, max(counts))
        table = [p + [self.spare[0] if self.spare else 0] * (width - len(p)) for p in self.ids]
        i32 = dict(dtype=torch.int32, device=device)
        self.table = torch.tensor(table, **i32)
        self.seq_lens = torch.tensor(self.lens, **i32)
        self.offsets = torch.tensor([0] + list(np.cumsum(self.new)), **i32)
        self.all_offsets = torch.tensor([0] + list(np.cumsum(self.lens)), **i32)
        self.rows, self.total = sum(self.new), sum(self.lens)
        self.pos = [p for n, m in zip(self.new, self.lens) for p in range(m - n, m)]

    def where(self):
        return self.offsets, self.seq_lens, self.table

    def whole(self):
        return self.all_offsets, self.seq_lens, self.table
