"""Workloads of the paged 4-bit KV cache, its attention, and token log probabilities.

Three operators of one serving step, each with a plain form in elementary torch
operations (``own = False``) and as a caller of mini_llama_b200 writes it
(``own = True``):

* append -- new keys and values of ragged sequences rotated to their positions,
  quantised to Q4_0 blocks and stored in a paged cache; the queries rotated in
  the same call; the stored rows read back as the values they stand for.
* attend -- causal attention of each sequence's last rows over its pages.
* logprobs -- log probability of given tokens, entropy, top alternatives.
"""
import math
import random

import torch

own = False

# ------------------------------------------------------------------ cases


def _append(name, seqs, new, ctx, ragged, heads, kv, hd, page, rope, theta, dtype, layout):
    return {"name": name, "op": "append", "seqs": seqs, "new": new, "ctx": ctx, "ragged": ragged,
            "heads": heads, "kv": kv, "hd": hd, "page": page, "rope": rope, "theta": theta,
            "dtype": dtype, "layout": layout}


def _attend(name, seqs, new, ctx, ragged, heads, kv, hd, page, dtype, layout):
    return {"name": name, "op": "attend", "seqs": seqs, "new": new, "ctx": ctx, "ragged": ragged,
            "heads": heads, "kv": kv, "hd": hd, "page": page, "dtype": dtype, "layout": layout}


def _logprobs(name, rows, vocab, top_k, dtype):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top_k": top_k,
            "dtype": dtype}


def listed():
    return [
        # one sequence's next token, llama3-8b heads: pure call latency
        _append("append_one", 1, 1, 512, False, 32, 8, 128, 16, "normal", 500000.0, "f32", 1),
        # one decode step of a full batch, qwen2-72b heads
        _append("append_batch", 64, 1, 4352, True, 64, 8, 128, 32, "neox", 1000000.0, "f32", 2),
        # prompts of uneven length prefilled together, llama3-8b heads
        _append("append_prompts", 5, 4096, 4096, True, 32, 8, 128, 64, "normal", 500000.0, "bf16",
                3),
        # one sequence's next token early in a chat: latency
        _attend("attend_one_short", 1, 1, 500, False, 32, 8, 128, 16, "f32", 4),
        # one sequence deep in a long document
        _attend("attend_one_long", 1, 1, 131072, False, 64, 8, 128, 64, "f32", 5),
        # a decode step of a full batch of uneven sequences, qwen2-72b heads
        _attend("attend_batch", 64, 1, 8192, True, 64, 8, 128, 16, "bf16", 6),
        # a few drafted tokens per sequence checked at once, llama2-7b heads (no sharing)
        _attend("attend_verify", 16, 5, 4096, True, 32, 32, 128, 32, "f32", 7),
        # a whole prompt, llama3-8b heads
        _attend("attend_prompt", 1, 4096, 4096, False, 32, 8, 128, 64, "bf16", 8),
        # uneven prompt chunks behind cached prefixes, the tiny model's odd head size
        _attend("attend_chunks", 5, 777, 2000, True, 6, 6, 48, 16, "f32", 9),
        # the next token's log probability and alternatives, llama3-8b vocabulary
        _logprobs("logprobs_one", 1, 128256, 20, "f32"),
        # a batch step, qwen2-72b vocabulary
        _logprobs("logprobs_batch", 64, 152064, 5, "f32"),
        # a prompt being scored, llama2-7b vocabulary
        _logprobs("logprobs_prompt", 4095, 32000, 1, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(32, 8, 128), (64, 8, 128), (32, 32, 128), (6, 6, 48), (8, 2, 64), (12, 4, 96),
          (16, 1, 128), (7, 7, 40), (4, 2, 32)]


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logprobs"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 152064)
        rows = _log_int(rng, 1, max(1, min(4095, 260000000 // _SIZE[dtype] // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab,
                "top_k": rng.choice([0, 1, 2, 5, 10, 20, 32]), "dtype": dtype}
    heads, kv, hd = rng.choice(_HEADS)
    page = rng.choice([16, 32, 48, 64, 128])
    layout = rng.randrange(1 << 30)
    if op == "append":
        seqs = _log_int(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, 5000 // seqs))
        ctx = max(new, _log_int(rng, 64, max(65, 131072 // seqs)))
        return {"op": op, "seqs": seqs, "new": new, "ctx": ctx, "ragged": True, "heads": heads,
                "kv": kv, "hd": hd, "page": page, "rope": rng.choice(["normal", "neox"]),
                "theta": rng.choice([10000.0, 500000.0, 1000000.0]), "dtype": dtype,
                "layout": layout}
    kind = rng.choice(["step", "verify", "prompt"])
    if kind == "prompt":
        new = _log_int(rng, 16, 2048)
        seqs = _log_int(rng, 1, max(1, 4096 // new))
        ctx = new + _log_int(rng, 1, 2048)
        seqs = max(1, min(seqs, int(1.3e11 / (4.0 * new * ctx * heads * hd))))
    else:
        seqs = _log_int(rng, 1, 64)
        new = 1 if kind == "step" else rng.randrange(2, 9)
        ctx = max(new, _log_int(rng, 16, 1048576 // (max(kv, 8) * seqs)))
    return {"op": op, "seqs": seqs, "new": new, "ctx": ctx, "ragged": True, "heads": heads,
            "kv": kv, "hd": hd, "page": page, "dtype": dtype, "layout": layout}


def _layout(case):
    """Per sequence: new rows, length after them, and its pages in the pool."""
    rng = random.Random(case["layout"])
    new, lens = [], []
    for _ in range(case["seqs"]):
        if case["ragged"]:
            n = rng.randrange((case["new"] + 1) // 2, case["new"] + 1)
            length = max(n, _log_int(rng, max(1, case["ctx"] // 16), case["ctx"]))
        else:
            n, length = case["new"], case["ctx"]
        new.append(n)
        lens.append(length)
    page = case["page"]
    counts = [(n + page - 1) // page for n in lens]
    ids = list(range(sum(counts) + 3))
    rng.shuffle(ids)
    pages, at = [], 0
    for c in counts:
        pages.append(ids[at:at + c])
        at += c
    return new, lens, pages, len(ids)


_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}


def work(case):
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top_k"]
        return {"bytes": n * v * _SIZE[case["dtype"]] + n * (12 + 8 * k), "flops": 4 * n * v}
    new, lens, _, _ = _layout(case)
    h, kv, hd, es = case["heads"], case["kv"], case["hd"], _SIZE[case["dtype"]]
    rows = sum(new)
    packed = kv * (hd // 2 + 2 * ((hd + 31) // 32)) * 2  # keys and values of one token
    if case["op"] == "append":
        # q, k, v in and q out; the packed rows written and read back; fp32 rows out
        return {"bytes": rows * ((2 * h + 2 * kv) * hd * es + 2 * packed + 2 * kv * hd * 4),
                "flops": rows * (h + 2 * kv) * hd * 6}
    seen = sum(n * length - n * (n - 1) // 2 for n, length in zip(new, lens))
    return {"bytes": rows * 2 * h * hd * es + sum(lens) * packed, "flops": 4 * seen * h * hd}


# ----------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=gen)


def _int32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _inputs_append(case, seed):
    gen = _gen(seed)
    new, lens, pages, n_pages = _layout(case)
    rows, t = sum(new), _TORCH[case["dtype"]]
    q = _randn(gen, rows, case["heads"], case["hd"]).to(t)
    k = (_randn(gen, rows, case["kv"], case["hd"]) * 2).to(t)
    v = _randn(gen, rows, case["kv"], case["hd"]).to(t)
    return new, lens, pages, n_pages, q, k, v


def _inputs_attend(case, seed):
    gen = _gen(seed)
    new, lens, pages, n_pages = _layout(case)
    rows, total = sum(new), sum(lens)
    # keys have a few strong channels, as rotated keys of real models do
    channel = 0.5 + torch.rand(case["kv"], case["hd"], device="cuda", generator=gen) * 1.5
    q = (_randn(gen, rows, case["heads"], case["hd"]) * 1.2).to(_TORCH[case["dtype"]])
    k = _randn(gen, total, case["kv"], case["hd"]) * channel
    v = _randn(gen, total, case["kv"], case["hd"])
    return new, lens, pages, n_pages, q, k, v


def _inputs_logprobs(case, seed):
    gen = _gen(seed)
    logits = (_randn(gen, case["rows"], case["vocab"]) * 2.5).to(_TORCH[case["dtype"]])
    tokens = torch.randint(case["vocab"], (case["rows"],), device="cuda", generator=gen,
                           dtype=torch.int32)
    return logits, tokens


# ------------------------------------------------------------ plain forms


def _half(x):
    """fp32 >= 0 to the nearest fp16 (halves up), kept in fp32."""
    normal = ((x.view(torch.int32) + 0x1000) >> 13 << 13).view(torch.float32)
    small = torch.floor(x.double() * 2.0 ** 24 + 0.5).float() * 2.0 ** -24
    r = torch.where(x < 2.0 ** -14, small, normal)
    return torch.where(r > 65504.0, torch.full_like(r, math.inf), r)


def _quantise(x):
    """Q4_0 codes (int8, minus 8) and fp32 block scales of the last axis of fp32 x."""
    hd = x.shape[-1]
    groups = (hd + 31) // 32
    b = torch.nn.functional.pad(x, (0, groups * 32 - hd)).unflatten(-1, (groups, 32))
    amax = b.abs().amax(-1)
    d = _half(amax / torch.full_like(amax, 7.0))
    inv = torch.where(d == 0, torch.zeros_like(d), torch.ones_like(d) / d)
    code = torch.floor((b * inv[..., None] + 8.0).double() + 0.5).clamp(0, 15) - 8
    return code.to(torch.int8).flatten(-2)[..., :hd], d


def _dequantise(code, d, hd):
    return code.float() * d.repeat_interleave(32, -1)[..., :hd]


def _rotate(x, pos, theta, rope):
    """x [rows, heads, hd] turned by its row's position, angles and products in 64 bits."""
    hd = x.shape[-1]
    j = torch.arange(hd // 2, device=x.device, dtype=torch.float64)
    angle = pos.double()[:, None] * torch.pow(torch.full_like(j, theta), -2.0 * j / hd)
    c, s = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    x = x.double()
    if rope == "neox":
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1).float()
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2).float()


def _positions(new, lens):
    return torch.cat([torch.arange(length - n, length, device="cuda")
                      for n, length in zip(new, lens)])


def _slots(counts, lens, pages, page):
    """Pool row of each sequence's last `counts` positions."""
    out = []
    for n, length, ids in zip(counts, lens, pages):
        pos = torch.arange(length - n, length, device="cuda")
        out.append(torch.tensor(ids, device="cuda")[pos // page] * page + pos % page)
    return torch.cat(out)


def _table(pages):
    width = max(1, max(len(p) for p in pages))
    return _int32([p + [0] * (width - len(p)) for p in pages])


class _Pool:
    """The plain cache: int8 codes and block scales, one row per token slot."""

    def __init__(self, slots, kv, hd):
        groups = (hd + 31) // 32
        self.kc = torch.zeros(slots, kv, hd, device="cuda", dtype=torch.int8)
        self.vc = torch.zeros_like(self.kc)
        self.kd = torch.zeros(slots, kv, groups, device="cuda")
        self.vd = torch.zeros_like(self.kd)


def _plain_append(st):
    case, pool, slots = st["case"], st["pool"], st["slots"]
    q = _rotate(st["q"], st["pos"], case["theta"], case["rope"]).to(st["q"].dtype)
    k = _rotate(st["k"], st["pos"], case["theta"], case["rope"])
    pool.kc[slots], pool.kd[slots] = _quantise(k)
    pool.vc[slots], pool.vd[slots] = _quantise(st["v"].float())
    hd = case["hd"]
    return (q, _dequantise(pool.kc[slots], pool.kd[slots], hd),
            _dequantise(pool.vc[slots], pool.vd[slots], hd))


def _plain_attend(st):
    case, pool, q = st["case"], st["pool"], st["q"]
    hd, kv = case["hd"], case["kv"]
    group = case["heads"] // kv
    out = torch.empty_like(q)
    row = 0
    for n, length, slots in zip(st["new"], st["lens"], st["slots"]):
        k = _dequantise(pool.kc[slots], pool.kd[slots], hd)  # [length, kv, hd]
        v = _dequantise(pool.vc[slots], pool.vd[slots], hd)
        x = q[row:row + n].float().view(n, kv, group, hd).permute(1, 2, 0, 3)
        s = x.reshape(kv, group * n, hd) @ k.permute(1, 2, 0) * (1.0 / math.sqrt(hd))
        s = s.view(kv, group, n, length)
        if n > 1:
            pos = torch.arange(length - n, length, device="cuda")
            hidden = torch.arange(length, device="cuda")[None, :] > pos[:, None]
            s = s.masked_fill(hidden, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = (p.view(kv, group * n, length) @ v.permute(1, 0, 2)).view(kv, group, n, hd)
        out[row:row + n] = o.permute(2, 0, 1, 3).reshape(n, case["heads"], hd).to(q.dtype)
        row += n
    return out


def _plain_logprobs(st):
    case, x = st["case"], st["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1)
    lse = m[:, 0] + torch.log(z)
    chosen = x.gather(1, st["tokens"].long()[:, None])[:, 0] - lse
    entropy = torch.log(z) - (e * (x - m)).sum(-1) / z
    # a stable sort keeps the lower index first among equal logits
    top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    k = case["top_k"]
    return (chosen, entropy, ids[:, :k].to(torch.int32).contiguous(),
            (top[:, :k] - lse[:, None]).contiguous())


# ------------------------------------------------------------------ calls


def prepare(case, seed):
    if case["op"] == "logprobs":
        logits, tokens = _inputs_logprobs(case, seed)
        return {"case": case, "logits": logits, "tokens": tokens}
    append = case["op"] == "append"
    new, lens, pages, n_pages, q, k, v = (_inputs_append if append else _inputs_attend)(case, seed)
    kv, hd, page = case["kv"], case["hd"], case["page"]
    st = {"case": case, "q": q, "new": new, "lens": lens}
    if append:
        st.update(k=k, v=v)
    if own:
        import mini_llama_b200 as mlb

        st["cache"] = mlb.CudaPagedKvCache(1, n_pages, page, kv, hd)
        st["offsets"], st["seq_lens"] = _int32(_offsets(new)), _int32(lens)
        st["table"] = _table(pages)
        st["rope"] = mlb.ROPE_NEOX if case.get("rope") == "neox" else mlb.ROPE_NORMAL
        if not append:
            st["cache"].AppendDevice(0, k, v, _int32(_offsets(lens)), st["seq_lens"], st["table"],
                                     rope_type=mlb.ROPE_NONE)
        return st
    st["pool"] = pool = _Pool(n_pages * page, kv, hd)
    if append:
        st["pos"], st["slots"] = _positions(new, lens), _slots(new, lens, pages, page)
        return st
    slots = _slots(lens, lens, pages, page)
    pool.kc[slots], pool.kd[slots] = _quantise(k)
    pool.vc[slots], pool.vd[slots] = _quantise(v)
    st["slots"] = list(slots.split(lens))
    return st


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend,
                "logprobs": _plain_logprobs}[case["op"]](state)
    import mini_llama_b200 as mlb

    if case["op"] == "logprobs":
        return mlb.CudaLogProbs(state["logits"], state["tokens"], top_k=case["top_k"])
    where = (state["offsets"], state["seq_lens"], state["table"])
    if case["op"] == "append":
        q = state["cache"].AppendDevice(0, state["k"], state["v"], *where, theta=case["theta"],
                                        rope_type=state["rope"], q=state["q"])
        k, v = state["cache"].ReadDevice(0, *where, q.shape[0])
        return q, k, v
    return mlb.CudaPagedAttentionDeviceInput(state["q"], state["cache"], 0, *where, case["heads"],
                                             case["kv"], case["hd"])


# ------------------------------------------------------------ definitions


def _exact_blocks(x):
    """Values Q4_0 keeps of fp32 rows, block by block: d is amax/7 as fp16 (halves
    up), the code the nearest of x/d + 8 (halves up) within 0..15. The code's
    fp32 steps belong to the format's definition."""
    out = torch.empty(x.shape, device=x.device, dtype=torch.float64)
    for at in range(0, x.shape[-1], 32):
        b = x[..., at:at + 32]
        top = b.abs().max(dim=-1, keepdim=True).values
        want = torch.div(top, torch.tensor(7.0, device=x.device).expand_as(top)).double()
        expo = torch.frexp(want)[1]
        step = torch.exp2((expo.double() - 11).clamp(min=-24.0))
        d = torch.floor(want / step + 0.5) * step
        d = torch.where(d > 65504.0, math.inf, d)
        inv = torch.where(d > 0, torch.ones_like(top) / d.float(), 0.0)
        y = (b * inv + 8.0).double()
        whole = y.trunc()
        code = torch.where(y - whole >= 0.5, whole + 1, whole).clamp(0.0, 15.0)
        out[..., at:at + 32] = (code - 8.0) * d
    return out


def _exact_append(case, seed):
    new, lens, _, _, q, k, v = _inputs_append(case, seed)
    pos = torch.cat([torch.arange(n, device="cuda") + (length - n)
                     for n, length in zip(new, lens)]).to(torch.float64)
    hd = case["hd"]
    half = hd // 2
    first = torch.arange(half, device="cuda") * (1 if case["rope"] == "neox" else 2)
    second = first + (half if case["rope"] == "neox" else 1)
    rate = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64)
                     * (-2.0 * math.log(case["theta"]) / hd))

    def turn(x):
        x = x.to(torch.float64)
        z = torch.complex(x[..., first], x[..., second])
        z = z * torch.polar(torch.ones_like(pos)[:, None], pos[:, None] * rate)[:, None, :]
        y = torch.empty_like(x)
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return turn(q), _exact_blocks(turn(k).to(torch.float32)), _exact_blocks(v.to(torch.float32))


def _exact_attend(case, seed):
    new, lens, _, _, q, k, v = _inputs_attend(case, seed)
    hd, kv, heads = case["hd"], case["kv"], case["heads"]
    k, v = _exact_blocks(k), _exact_blocks(v)
    out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    row = start = 0
    for n, length in zip(new, lens):
        for h in range(heads):
            kh = k[start:start + length, h * kv // heads]
            vh = v[start:start + length, h * kv // heads]
            s = torch.einsum("id,td->it", q[row:row + n, h].double(), kh) / math.sqrt(hd)
            last = torch.arange(length - n, length, device="cuda")[:, None]
            s = torch.where(torch.arange(length, device="cuda")[None] <= last, s, -math.inf)
            out[row:row + n, h] = torch.einsum("it,td->id", torch.softmax(s, -1), vh)
        row, start = row + n, start + length
    return out


def _exact_logprobs(case, seed):
    logits, tokens = _inputs_logprobs(case, seed)
    n, k = case["rows"], case["top_k"]
    chosen = torch.empty(n, device="cuda", dtype=torch.float64)
    entropy = torch.empty_like(chosen)
    ids = torch.empty(n, k, device="cuda", dtype=torch.int32)
    top = torch.empty(n, k, device="cuda", dtype=torch.float64)
    for r in range(0, n, 512):
        x = logits[r:r + 512].double()
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        chosen[r:r + 512] = lp[torch.arange(len(lp), device="cuda"), tokens[r:r + 512].long()]
        entropy[r:r + 512] = -(lp.exp() * lp).sum(-1)
        for j in range(k):
            # the lowest index among the largest left
            best = x.max(-1, keepdim=True).values
            at = (x == best).to(torch.int8).argmax(-1, keepdim=True)
            ids[r:r + 512, j] = at[:, 0].to(torch.int32)
            top[r:r + 512, j] = lp.gather(1, at)[:, 0]
            x.scatter_(1, at, -math.inf)
    return chosen, entropy, ids, top


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend,
            "logprobs": _exact_logprobs}[case["op"]](case, seed)
