"""The int8 layer's operators in 64 bits (torch, any device)."""
import math

import torch


def to_codes(t, root=None):
    """Codes (int8) and scales (float64) of rows of values t (float64)."""
    top = t.abs().amax(-1, keepdim=True)
    code = torch.where(top > 0, torch.round(t * 127.0 / top), torch.zeros_like(t))
    scale = top[:, 0] / 127.0
    if root is not None:
        scale = torch.where(top[:, 0] > 0, scale * root, torch.zeros_like(scale))
    return code.nan_to_num(0.0).to(torch.int8), scale


def norm_codes(h, w, eps):
    h = h.double()
    root = 1.0 / torch.sqrt((h * h).mean(-1) + float(torch.tensor(eps, dtype=torch.float32)))
    return to_codes(h * w.double(), root)


def silu_mul(g, u):
    g = g.double()
    return g / (1.0 + torch.exp(-g)) * u.double()


def linear(x, sx, w, sw, bias=None):
    """y and what its rounding errors are relative to."""
    total = x.double() @ w.double().t()
    y = total * sx.double()[:, None] * sw.double()
    size = y.abs()
    if bias is not None:
        y = y + bias.double()
    return y, size


def frequencies(rot, theta, scaling="none", factor=1.0, trained=0.0, low=1.0, high=4.0, fast=32.0,
                slow=1.0):
    out, gain = [], 1.0
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "llama3":
            wave = 2.0 * math.pi / f
            if wave > trained / low:
                f /= factor
            elif wave > trained / high:
                keep = (trained / wave - low) / (high - low)
                f = (1.0 - keep) * f / factor + keep * f
        elif scaling == "yarn":
            def pair(turns):
                return rot * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

            a, b = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
            ramp = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            f = ramp * f / factor + (1.0 - ramp) * f
            gain = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
        out.append(f)
    return torch.tensor(out, dtype=torch.float64), gain


def rope(x, pos, f, gain, neox):
    """x [rows, heads, dim] turned in its first 2 len(f) dimensions."""
    half = len(f)
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
    angle = pos.double()[:, None] * f.to(x.device)
    c, s = (gain * torch.cos(angle))[:, None], (gain * torch.sin(angle))[:, None]
    y = x.double()
    p, q = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = p * c - q * s, p * s + q * c
    return y
