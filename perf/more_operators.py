"""Workloads of a transformer layer in 8-bit integers: norm, product, rotation, activation.

Four operators of one layer over rows of many sequences, each with a plain form
in elementary torch operations (``own = False``) and as a caller of
mini_llama_b200 writes it (``own = True``):

* norm -- the residual's addition, RMSNorm, and the row as int8 codes with one scale.
* linear -- product of int8 codes with a scale for each token and each channel.
* rope -- queries and keys turned to their rows' positions: interleaved and half
  layouts, part of the head, frequencies scaled for long contexts.
* silu -- SiLU(gate) * up, and the row as int8 codes with one scale.

Codes are returned as the values that they stand for.
"""
import math

import torch

own = False

# ------------------------------------------------------------------ cases


def _norm(name, rows, n, residual, dtype, eps):
    return {"name": name, "op": "norm", "rows": rows, "n": n, "residual": residual,
            "dtype": dtype, "eps": eps}


def _linear(name, rows, k, n, bias, dtype):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "bias": bias,
            "dtype": dtype}


def _silu(name, rows, n, dtype):
    return {"name": name, "op": "silu", "rows": rows, "n": n, "dtype": dtype}


def _rope(name, rows, far, heads, kv, hd, rot, layout, theta, scaling, dtype):
    return {"name": name, "op": "rope", "rows": rows, "far": far, "heads": heads, "kv": kv,
            "hd": hd, "rot": rot, "layout": layout, "theta": theta, "scaling": scaling,
            "dtype": dtype}


def listed():
    return [
        # one sequence's next token, llama3-8b width: call latency
        _norm("norm_one", 1, 4096, True, "f32", 1e-5),
        # a decode step of a full batch, qwen2-72b width
        _norm("norm_batch", 64, 8192, True, "f32", 1e-6),
        # a prompt, qwen2-72b width
        _norm("norm_prompt", 4096, 8192, True, "bf16", 1e-6),
        # one sequence's next token, llama2-7b output projection
        _linear("linear_one", 1, 4096, 4096, False, "f32"),
        # a decode step of a batch, qwen2-72b query, key and value projection
        _linear("linear_batch", 32, 8192, 10240, True, "f32"),
        # prompts of uneven length one after another, the tiny model's odd sizes
        _linear("linear_ragged", 777, 288, 1536, True, "bf16"),
        # a prompt, llama3-8b gate and up projection
        _linear("linear_prompt", 4096, 4096, 28672, False, "bf16"),
        # one sequence's next token, llama3-8b heads, long-context frequencies
        _rope("rope_one", 1, 131072, 32, 8, 128, 128, "normal", 500000.0, "llama3", "f32"),
        # a decode step of a batch, qwen2-72b heads
        _rope("rope_batch", 64, 131072, 64, 8, 128, 128, "neox", 1000000.0, "yarn", "f32"),
        # a prompt, llama3-8b heads, half of each head turned
        _rope("rope_prompt", 4096, 16384, 32, 8, 128, 64, "neox", 500000.0, "linear", "bf16"),
        # a decode step of a batch, qwen2-72b hidden width
        _silu("silu_batch", 64, 29568, "f32"),
        # a prompt, llama3-8b hidden width
        _silu("silu_prompt", 4096, 14336, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(32, 8, 128), (64, 8, 128), (32, 32, 128), (6, 6, 48), (8, 2, 64), (12, 4, 96),
          (16, 1, 128), (7, 7, 40), (4, 2, 32)]


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "rope", "silu"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "norm":
        n = _log_int(rng, 64, 8192)
        rows = _log_int(rng, 1, min(4096, 16000000 // n))
        return {"op": op, "rows": rows, "n": n, "residual": rng.random() < 0.7, "dtype": dtype,
                "eps": rng.choice([1e-5, 1e-6])}
    if op == "linear":
        k = _log_int(rng, 64, 29568)
        n = _log_int(rng, 64, min(28672, 250000000 // k))
        rows = _log_int(rng, 1, max(1, min(4096, int(4.8e11 / (k * n)))))
        return {"op": op, "rows": rows, "k": k, "n": n, "bias": rng.random() < 0.5,
                "dtype": dtype}
    if op == "silu":
        n = _log_int(rng, 64, 29568)
        return {"op": op, "rows": _log_int(rng, 1, min(4096, 29000000 // n)), "n": n,
                "dtype": dtype}
    heads, kv, hd = rng.choice(_HEADS)
    return {"op": op, "rows": _log_int(rng, 1, 4096), "far": _log_int(rng, 64, 131072),
            "heads": heads, "kv": kv, "hd": hd, "rot": hd // rng.choice([1, 1, 2, 4]) // 2 * 2,
            "layout": rng.choice(["normal", "neox"]),
            "theta": rng.choice([10000.0, 500000.0, 1000000.0]),
            "scaling": rng.choice(["none", "linear", "llama3", "yarn"]), "dtype": dtype}


_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}


def work(case):
    es, rows = _SIZE[case["dtype"]], case["rows"]
    if case["op"] == "norm":
        # x (and the residual) in, the values in fp32 (and the sum) out
        n = case["n"]
        return {"bytes": rows * n * (es * (3 if case["residual"] else 1) + 4) + 4 * n,
                "flops": 8 * rows * n}
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        return {"bytes": (rows + n) * (k + 4) + rows * n * es + (4 * n if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    if case["op"] == "silu":
        return {"bytes": rows * case["n"] * (2 * es + 4), "flops": 8 * rows * case["n"]}
    values = rows * (case["heads"] + case["kv"]) * case["hd"]
    return {"bytes": 2 * values * es + 4 * rows, "flops": 3 * values}


# ----------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=gen)


def _inputs_norm(case, seed):
    gen = _gen(seed)
    rows, n, t = case["rows"], case["n"], _TORCH[case["dtype"]]
    # a residual stream has a few strong channels; a norm's weights lie around 1
    channel = torch.exp(_randn(gen, n) * 0.6)
    x = (_randn(gen, rows, n) * channel).to(t)
    r = (_randn(gen, rows, n) * 0.5).to(t) if case["residual"] else None
    return x, r, 1.0 + 0.2 * _randn(gen, n)


def _codes(gen, rows, n):
    """int8 codes of rows of normal values, each row 16-byte aligned."""
    padded = torch.zeros(rows, (n + 15) // 16 * 16, device="cuda", dtype=torch.int8)
    padded[:, :n] = (_randn(gen, rows, n) * 34.0).round().clamp(-127, 127).to(torch.int8)
    return padded[:, :n]


def _inputs_linear(case, seed):
    gen = _gen(seed)
    x, w = _codes(gen, case["rows"], case["k"]), _codes(gen, case["n"], case["k"])
    sx = 0.01 + 0.05 * torch.rand(case["rows"], device="cuda", generator=gen)
    sw = 0.0004 + 0.0006 * torch.rand(case["n"], device="cuda", generator=gen)
    bias = _randn(gen, case["n"]) * 0.5 if case["bias"] else None
    return x, sx, w, sw, bias


def _inputs_silu(case, seed):
    # gate and up as one product leaves them, side by side
    both = (_randn(_gen(seed), case["rows"], 2 * case["n"]) * 1.5).to(_TORCH[case["dtype"]])
    return both[:, :case["n"]], both[:, case["n"]:]


def _inputs_rope(case, seed):
    gen = _gen(seed)
    t = _TORCH[case["dtype"]]
    q = _randn(gen, case["rows"], case["heads"], case["hd"]).to(t)
    k = (_randn(gen, case["rows"], case["kv"], case["hd"]) * 2).to(t)
    pos = torch.randint(case["far"], (case["rows"],), device="cuda", generator=gen,
                        dtype=torch.int32)
    return q, k, pos


# parameters of scaled frequencies as checkpoints state them
_SCALE, _TRAINED, _LOW, _HIGH, _FAST, _SLOW = 8.0, 8192, 1.0, 4.0, 32.0, 1.0

# ------------------------------------------------------------ plain forms


def _to_codes(t, factor=None):
    """Values that int8 codes of rows t (64 bits) stand for, in fp32; factor is what
    of each row's values is left out of t."""
    top = t.abs().amax(-1, keepdim=True)
    # values next to a code's border: 64 bits
    code = torch.where(top > 0, torch.round(t * 127.0 / top), torch.zeros_like(t))
    scale = top / 127.0 if factor is None else top * factor / 127.0
    return code.float() * scale.float()


def _plain_norm(st):
    x, r, w, eps = st["x"], st["r"], st["w"], st["case"]["eps"]
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    y = h.double()
    root = 1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    values = _to_codes(y * w.double(), root)
    return values if r is None else (values, h)


def _plain_linear(st):
    x, w = st["x"], st["w"]
    # sums of 1024 products of codes are whole numbers below 2^24: exact in fp32
    total = torch.zeros(x.shape[0], w.shape[0], device=x.device, dtype=torch.float64)
    for at in range(0, x.shape[1], 1024):
        total += x[:, at:at + 1024].float() @ w[:, at:at + 1024].float().t()
    y = total.float() * st["sx"][:, None] * st["sw"][None, :]
    if st["bias"] is not None:
        y = y + st["bias"]
    return y.to(_TORCH[st["case"]["dtype"]])


def _plain_silu(st):
    g = st["gate"].double()
    return _to_codes(g / (1.0 + torch.exp(-g)) * st["up"].double())


def _frequencies(case):
    """Angles per position of each pair, and the factor of cosine and sine."""
    rot, theta = case["rot"], case["theta"]
    j = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    f = torch.pow(torch.full_like(j, theta), -2.0 * j / rot)
    if case["scaling"] == "none":
        return f, 1.0
    if case["scaling"] == "linear":
        return f / _SCALE, 1.0
    if case["scaling"] == "llama3":
        turns = _TRAINED * f / (2.0 * math.pi)  # over the trained length
        keep = ((turns - _LOW) / (_HIGH - _LOW)).clamp(0.0, 1.0)
        return f / _SCALE * (1.0 - keep) + f * keep, 1.0

    def pair(turns):
        return rot * math.log(_TRAINED / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

    first = max(math.floor(pair(_FAST)), 0)
    last = min(math.ceil(pair(_SLOW)), rot - 1)
    ramp = ((j - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
    return f / _SCALE * ramp + f * (1.0 - ramp), 0.1 * math.log(_SCALE) + 1.0


def _plain_rope(st):
    case, f = st["case"], st["frequencies"]
    rot = case["rot"]
    angle = st["pos"].double()[:, None] * f  # positions are far: 64 bits
    c = (torch.cos(angle) * st["factor"]).float()[:, None, :]
    s = (torch.sin(angle) * st["factor"]).float()[:, None, :]

    def turn(x):
        y = x.float()
        head, rest = y[..., :rot], y[..., rot:]
        if case["layout"] == "neox":
            a, b = head[..., :rot // 2], head[..., rot // 2:]
            head = torch.cat([a * c - b * s, a * s + b * c], -1)
        else:
            a, b = head[..., 0::2], head[..., 1::2]
            head = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
        return torch.cat([head, rest], -1).to(x.dtype)

    return turn(st["q"]), turn(st["k"])


# ------------------------------------------------------------------ calls


def prepare(case, seed):
    st = {"case": case}
    if case["op"] == "norm":
        st["x"], st["r"], st["w"] = _inputs_norm(case, seed)
    elif case["op"] == "linear":
        st["x"], st["sx"], st["w"], st["sw"], st["bias"] = _inputs_linear(case, seed)
    elif case["op"] == "silu":
        st["gate"], st["up"] = _inputs_silu(case, seed)
    else:
        st["q"], st["k"], st["pos"] = _inputs_rope(case, seed)
        if own:
            import mini_llama_b200 as mlb

            st["table"] = mlb.RopeTable(
                case["rot"], case["theta"],
                scaling={"none": mlb.ROPE_SCALING_NONE, "linear": mlb.ROPE_SCALING_LINEAR,
                         "llama3": mlb.ROPE_SCALING_LLAMA3,
                         "yarn": mlb.ROPE_SCALING_YARN}[case["scaling"]],
                factor=_SCALE, original_len=_TRAINED, low_freq_factor=_LOW,
                high_freq_factor=_HIGH, beta_fast=_FAST, beta_slow=_SLOW)
            st["layout"] = mlb.ROPE_NEOX if case["layout"] == "neox" else mlb.ROPE_NORMAL
        else:
            st["frequencies"], st["factor"] = _frequencies(case)
    return st


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "silu": _plain_silu,
                "rope": _plain_rope}[op](state)
    import mini_llama_b200 as mlb

    if op == "norm":
        eps = state["case"]["eps"]
        if state["r"] is None:
            return mlb.CudaInt8DequantizeDeviceInput(
                *mlb.CudaRmsNormInt8DeviceWeight(state["x"], state["w"], eps))
        codes, scale, h = mlb.CudaRmsNormInt8DeviceWeight(state["x"], state["w"], eps,
                                                          residual=state["r"])
        return mlb.CudaInt8DequantizeDeviceInput(codes, scale), h
    if op == "linear":
        return mlb.CudaInt8LinearDeviceInput(state["x"], state["sx"], state["w"], state["sw"],
                                             bias=state["bias"],
                                             out_dtype=_TORCH[state["case"]["dtype"]])
    if op == "silu":
        return mlb.CudaInt8DequantizeDeviceInput(
            *mlb.CudaSiluMulInt8DeviceInput(state["gate"], state["up"]))
    return mlb.CudaRopeRowsDeviceInput(state["q"], state["k"], state["pos"], state["table"],
                                       rope_type=state["layout"])


# ------------------------------------------------------------ definitions


def _exact_codes(t, factor):
    """Row by row: 127 steps from 0 to the largest magnitude, the nearest step (even
    on ties), and what it stands for."""
    largest = t.abs().max(dim=-1, keepdim=True).values
    live = largest > 0
    steps = torch.div(127.0 * t, torch.where(live, largest, torch.ones_like(largest)))
    low = torch.floor(steps)
    part = steps - low
    odd = torch.remainder(low, 2.0) == 1.0
    code = torch.where((part > 0.5) | ((part == 0.5) & odd), low + 1.0, low)
    return code * (largest / 127.0) * factor


def _exact_norm(case, seed):
    x, r, w = _inputs_norm(case, seed)
    if r is not None:
        full = x.to(torch.float64) + r.to(torch.float64)
        h = full.to(torch.float32).to(x.dtype).to(torch.float64)
    else:
        h = x.to(torch.float64)
    power = torch.linalg.vector_norm(h, dim=-1, keepdim=True) ** 2 / case["n"]
    values = _exact_codes(h * w.to(torch.float64), torch.rsqrt(power + case["eps"]))
    return values if r is None else (values, full)


def _exact_linear(case, seed):
    x, sx, w, sw, bias = _inputs_linear(case, seed)
    out = torch.empty(case["rows"], case["n"], device="cuda", dtype=torch.float64)
    xd = x.to(torch.float64)
    for at in range(0, case["n"], 4096):
        # whole numbers below 2^53
        out[:, at:at + 4096] = torch.einsum("mk,nk->mn", xd, w[at:at + 4096].to(torch.float64))
    out *= sx.to(torch.float64)[:, None]
    out *= sw.to(torch.float64)
    return out if bias is None else out.add_(bias.to(torch.float64))


def _exact_silu(case, seed):
    gate, up = _inputs_silu(case, seed)
    g = gate.to(torch.float64)
    return _exact_codes(g * torch.sigmoid(g) * up.to(torch.float64), 1.0)


def _exact_rope(case, seed):
    q, k, pos = _inputs_rope(case, seed)
    rot = case["rot"]
    half = rot // 2
    rates, gain = [], 1.0
    for i in range(half):
        rate = math.exp(-2.0 * i / rot * math.log(case["theta"]))
        slow = rate / _SCALE
        if case["scaling"] == "linear":
            rate = slow
        elif case["scaling"] == "llama3":
            wave = 2.0 * math.pi / rate
            if wave > _TRAINED / _LOW:
                rate = slow
            elif wave >= _TRAINED / _HIGH:
                mix = (_TRAINED / wave - _LOW) / (_HIGH - _LOW)
                rate = (1.0 - mix) * slow + mix * rate
        elif case["scaling"] == "yarn":
            ends = [rot / 2.0 * math.log(_TRAINED / (2.0 * math.pi * turns))
                    / math.log(case["theta"]) for turns in (_FAST, _SLOW)]
            lo, hi = max(0, math.floor(ends[0])), min(rot - 1, math.ceil(ends[1]))
            mix = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            rate = mix * slow + (1.0 - mix) * rate
            gain = 1.0 + 0.1 * math.log(_SCALE)
        rates.append(rate)
    neox = case["layout"] == "neox"
    first = torch.arange(half, device="cuda") * (1 if neox else 2)
    second = first + (half if neox else 1)
    angle = pos.to(torch.float64)[:, None] * torch.tensor(rates, device="cuda",
                                                          dtype=torch.float64)
    spin = torch.polar(torch.full_like(angle, gain), angle)[:, None, :]

    def turn(x):
        y = x.to(torch.float64)
        z = torch.complex(y[..., first], y[..., second]) * spin
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return turn(q), turn(k)


def exact(case, seed):
    return {"norm": _exact_norm, "linear": _exact_linear, "silu": _exact_silu,
            "rope": _exact_rope}[case["op"]](case, seed)
