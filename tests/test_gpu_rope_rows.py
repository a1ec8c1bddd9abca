"""RoPE of rows at positions of their own, against 64 bits.

The angle's turns, below 2^31 / 2 pi, are off by 2^-52 of themselves, so by 2^-24 of a
turn at the farthest and less than 2^-36 below 2^17; rounded to fp32 (half a turn at most)
by 2^-25, sine and cosine by 2 ulp (2^-22) and the amplitude by 2^-24, the two products
and their sum by 2^-24 each: below (pi 2^-24 + 2^-22 + 4 2^-24) = 12 2^-24 of |a| + |b|.
bf16 adds 2^-8 of the result.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import int8_ref as ref  # noqa: E402

U = 2.0 ** -24
KINDS = {"none": 0, "linear": 1, "llama3": 2, "yarn": 3}


def table(rot, theta, scaling):
    args = dict(factor=8.0, trained=8192.0)
    t = mlb.RopeTable(rot, theta, KINDS[scaling], factor=8.0, original_len=8192)
    f, gain = ref.frequencies(rot, theta, scaling, **args)
    # two ways to the same numbers, each a few 64-bit roundings long
    assert torch.allclose(t.frequencies.cpu(), f, rtol=1e-14, atol=0) and math.isclose(
        t.amplitude, gain, rel_tol=1e-15)
    return t, t.frequencies.cpu(), gain


def check(got, x, pos, f, gain, neox, far=0.0):
    want = ref.rope(x, pos, f, gain, neox)
    half = len(f)
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
    size = torch.zeros_like(want)
    size[..., a] = size[..., b] = gain * (x.double()[..., a].abs() + x.double()[..., b].abs())
    tol = (12 * U + far) * size
    if x.dtype is torch.bfloat16:
        tol = tol + 2.0 ** -8 * want.abs()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err - tol).max()
    assert torch.equal(got[..., 2 * half:], x[..., 2 * half:])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("rows,heads,kv,dim,rot,scaling", [
    (1, 32, 8, 128, 128, "none"), (64, 64, 8, 128, 128, "yarn"), (300, 32, 8, 128, 64, "linear"),
    (5, 6, 6, 48, 48, "llama3"), (7, 7, 7, 40, 10, "none"), (3, 1, 1, 2, 2, "none"),
    (9, 12, 4, 96, 24, "yarn"), (2, 3, 1, 256, 250, "llama3"), (2, 2, 2, 1024, 1024, "linear"),
    (4, 5, 3, 22, 6, "yarn"), (2000, 4, 2, 64, 32, "llama3")])
def test_rope(cuda, rows, heads, kv, dim, rot, scaling, neox, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + dim + rot)
    t = getattr(torch, dtype)
    q = torch.randn(rows, heads, dim, device="cuda", generator=g).to(t)
    k = torch.randn(rows, kv, dim, device="cuda", generator=g).to(t)
    pos = torch.randint(131072, (rows,), device="cuda", generator=g, dtype=torch.int32)
    tab, f, gain = table(rot, 500000.0, scaling)
    kind = mlb.ROPE_NEOX if neox else mlb.ROPE_NORMAL
    q_out, k_out = mlb.CudaRopeRowsDeviceInput(q, k, pos, tab, rope_type=kind)
    check(q_out, q, pos, f, gain, neox)
    check(k_out, k, pos, f, gain, neox)
    # in place, alone, and inside one product's rows
    q2 = q.clone()
    assert mlb.CudaRopeRowsDeviceInput(q2, None, pos, tab, kind, q_out=q2) == (q2, None)
    assert torch.equal(q2, q_out)
    one = mlb.CudaRopeRowsDeviceInput(None, k, pos, tab, kind)
    assert one[0] is None and torch.equal(one[1], k_out)
    both = torch.randn(rows, (heads + 2 * kv) * dim, device="cuda", generator=g).to(t)
    qv = both[:, :heads * dim].view(rows, heads, dim)
    kv_ = both[:, heads * dim:(heads + kv) * dim].view(rows, kv, dim)
    qv.copy_(q), kv_.copy_(k)
    v = both[:, (heads + kv) * dim:].clone()
    mlb.CudaRopeRowsDeviceInput(qv, kv_, pos, tab, kind, q_out=qv, k_out=kv_)
    assert torch.equal(qv, q_out) and torch.equal(kv_, k_out)
    assert torch.equal(both[:, (heads + kv) * dim:], v)


@pytest.mark.parametrize("neox", [False, True])
def test_unaligned_rows(cuda, neox):
    g = torch.Generator(device="cuda").manual_seed(4)
    for t in (torch.float32, torch.bfloat16):
        flat = torch.randn(9 * 131 + 1, device="cuda", generator=g).to(t)
        x = flat[1:].view(9, 131)[:, :128].view(9, 2, 64)
        pos = torch.arange(9, device="cuda", dtype=torch.int32)
        tab, f, gain = table(32, 10000.0, "none")
        out, _ = mlb.CudaRopeRowsDeviceInput(x, None, pos, tab, int(neox))
        check(out, x, pos, f, gain, neox)


def test_any_position(cuda):
    """Zero, negative and the farthest positions."""
    pos = torch.tensor([0, -1, -131071, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(5, 3, 64, device="cuda", generator=g)
    tab, f, gain = table(64, 10000.0, "none")
    out, _ = mlb.CudaRopeRowsDeviceInput(x, None, pos, tab)
    # the frequency over 2 pi, the product: 2^-52 of 2^31 / 2 pi turns, in radians 2^-21;
    # the 64-bit form's own product 2^-53 of 2^31
    check(out, x, pos, f, gain, False, far=2.0 ** -20)
    assert torch.equal(out[0], x[0])


def test_factors_of_a_checkpoint(cuda):
    fac = np.linspace(1.0, 8.0, 16)
    tab = mlb.RopeTable(32, 10000.0, factors=fac)
    f = ref.frequencies(32, 10000.0)[0].numpy() / fac
    assert np.allclose(tab.frequencies.cpu().numpy(), f, rtol=1e-14, atol=0)


def test_agrees_with_the_one_row_form(cuda):
    """mlb_rope's fp32 angles differ by up to pos 2^-24 (twice that through 10000^x)."""
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(1, 8, 64, device="cuda", generator=g)
    k = torch.randn(1, 2, 64, device="cuda", generator=g)
    for kind in (0, 1):
        q1, k1 = q.clone().view(-1), k.clone().view(-1)
        mlb.CudaRopeDeviceInput(q1, k1, 8, 2, 64, 77, 10000.0, kind)
        a, b = mlb.CudaRopeRowsDeviceInput(q, k, torch.tensor([77], dtype=torch.int32, device="cuda"),
                                           mlb.RopeTable(64), kind)
        tol = (4 * 77 + 16) * U * 8
        assert (a.view(-1) - q1).abs().max() < tol and (b.view(-1) - k1).abs().max() < tol


def test_no_rows_and_non_finite_values(cuda):
    tab = mlb.RopeTable(64)
    e = torch.empty(0, 3, 64, device="cuda")
    out, _ = mlb.CudaRopeRowsDeviceInput(e, None, torch.empty(0, dtype=torch.int32, device="cuda"), tab)
    assert out.shape == e.shape
    x = torch.ones(2, 1, 64, device="cuda")
    x[0, 0, 4] = math.nan
    out, _ = mlb.CudaRopeRowsDeviceInput(x, None, torch.tensor([3, 3], dtype=torch.int32, device="cuda"), tab)
    bad = torch.isnan(out)
    assert bad[0, 0, 4:6].all() and int(bad.sum()) == 2


def test_replaced_frequencies(cuda):
    """What stands in a table's place of frequencies is read in every form, or refused."""
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(3, 2, 64, device="cuda", generator=g)
    k = torch.randn(3, 1, 64, device="cuda", generator=g)
    pos = torch.tensor([5, 900, 131071], dtype=torch.int32, device="cuda")
    tab = mlb.RopeTable(64)
    f = ref.frequencies(32, 500000.0)[0]
    tab.frequencies = f.cuda()
    q_out, k_out = mlb.CudaRopeRowsDeviceInput(q, k, pos, tab)
    check(q_out, q, pos, f, 1.0, False)
    check(k_out, k, pos, f, 1.0, False)
    alone, _ = mlb.CudaRopeRowsDeviceInput(q, None, pos, tab)
    assert torch.equal(alone, q_out)
    for bad in (f.float().cuda(), f.cuda()[None], f.cuda()[::2], f):
        tab.frequencies = bad
        with pytest.raises(mlb.MlbError, match="frequencies"):
            mlb.CudaRopeRowsDeviceInput(q, k, pos, tab)
        with pytest.raises(mlb.MlbError, match="frequencies"):
            mlb.CudaRopeRowsDeviceInput(q, None, pos, tab)
