"""Rows as int8 codes: as they are, after RMSNorm, after SiLU(gate) * up, and back.

Codes are the 64-bit form's, every one. Scales: A / 127 (times the root) rounded once;
the root's sum of squares is fp32, up to 40 terms one after another in a thread and a
tree of at most 42 more steps (5 in a warp, 32 warps, 5 again), each off by 2^-24, half
of which the square root passes on: below 45 * 2^-24 together.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import int8_ref as ref  # noqa: E402

U = 2.0 ** -24
TYPES = ["float32", "bfloat16"]
SHAPES = [(1, 1), (3, 7), (5, 32), (2, 100), (64, 288), (7, 777), (33, 1024), (1, 4096),
          (300, 4096), (5, 8192), (700, 1000), (4, 11008), (3, 29568), (2, 32768), (2, 40001)]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def check(got, want, tol=U):
    codes, scales = got[:2]
    assert codes.dtype is torch.int8 and scales.dtype is torch.float32
    assert torch.equal(codes, want[0]), (codes != want[0]).sum()
    err = (scales.double() - want[1]).abs()
    # below fp32's normal numbers a scale is rounded to the smallest step
    assert (err <= want[1] * tol + 2.0 ** -150).all(), (err / want[1]).max() / U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_quantize(cuda, rows, n, dtype):
    x = (randn(gen(rows * n), rows, n) * 3).to(getattr(torch, dtype))
    got = mlb.CudaInt8QuantizeDeviceInput(x)
    check(got, ref.to_codes(x.double()))
    assert got[0].stride(0) % 16 == 0 and got[0].data_ptr() % 16 == 0
    again = mlb.CudaInt8QuantizeDeviceInput(x)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    for out in TYPES:
        back = mlb.CudaInt8DequantizeDeviceInput(*got, out_dtype=getattr(torch, out))
        want = (got[0].float() * got[1][:, None]).to(getattr(torch, out))
        assert torch.equal(back, want)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_norm(cuda, rows, n, dtype, residual):
    g = gen(rows + n)
    t = getattr(torch, dtype)
    x, w = randn(g, rows, n).to(t), 1 + 0.3 * randn(g, n)
    r = (randn(g, rows, n) * 2).to(t) if residual else None
    got = mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=r)
    h = x
    if residual:
        h = (x.float() + r.float()).to(t)
        assert torch.equal(got[2], h)
    check(got, ref.norm_codes(h, w, 1e-5), 45 * U)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_silu_mul(cuda, rows, n, dtype):
    both = (randn(gen(rows + 3 * n), rows, 2 * n) * 2.5).to(getattr(torch, dtype))
    gate, up = both[:, :n], both[:, n:]
    check(mlb.CudaSiluMulInt8DeviceInput(gate, up), ref.to_codes(ref.silu_mul(gate, up)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [96, 1000, 4099])
def test_rows_of_any_kind(cuda, n, dtype):
    """Zero rows, one value alone, tiny, subnormal and huge rows, values on codes'
    borders; with NaN or an infinity: scale NaN, the other rows as ever."""
    t = getattr(torch, dtype)
    x = randn(gen(n), 14, n)
    x[0] = 0.0
    x[1] = 0.0
    x[1, n // 2] = -5.0
    x[2] *= 1e-33
    x[3] *= 1e-39
    x[4] = x[4].clamp(-3, 3) * 1e38
    x[5] = (torch.arange(n, device="cuda") % 255 - 127) * 2.0  # A = 254: halves are exact
    x[6] = x[5] * 0.5 + 0.25
    x[6, 0] = 254.0
    x[7, 3] = math.nan
    x[8, n - 1] = math.inf
    x[9, 0] = -math.inf
    x[10] = 1.0
    x[11] = -0.0
    x[12] *= 1e18
    x[13] *= 1e-18
    x = x.to(t)
    ok = torch.tensor([i not in (7, 8, 9) for i in range(14)], device="cuda")
    w = 1 + 0.2 * randn(gen(n + 1), n)
    w[1] = 0.0
    one = torch.ones(n, device="cuda")
    silu = ref.silu_mul(x, x.flip(1))
    for got, want, tol in (
            (mlb.CudaInt8QuantizeDeviceInput(x), ref.to_codes(x.double()), U),
            (mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-6), ref.norm_codes(x, w, 1e-6), 45 * U),
            (mlb.CudaRmsNormInt8DeviceWeight(x, one, 0.0), ref.norm_codes(x, one, 0.0), 45 * U)):
        check((got[0][ok], got[1][ok]), (want[0][ok], want[1][ok]), tol)
        assert torch.isnan(got[1][~ok]).all()
        assert torch.isnan(mlb.CudaInt8DequantizeDeviceInput(*got)[~ok]).all()
    got, want = mlb.CudaSiluMulInt8DeviceInput(x, x.flip(1)), ref.to_codes(silu)
    whole = torch.isfinite(silu).all(-1) & (want[1] < 3e38)
    check((got[0][whole], got[1][whole]), (want[0][whole], want[1][whole]))
    assert torch.isnan(got[1][~whole]).all()
    r = torch.zeros_like(x)
    codes, scales, s = mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-6, residual=r)
    want = ref.norm_codes(x, w, 1e-6)
    check((codes[ok], scales[ok]), (want[0][ok], want[1][ok]), 45 * U)
    assert torch.equal(s[ok], x[ok]) and torch.isnan(scales[~ok]).all()


@pytest.mark.parametrize("gate", [-200.0, -95.0, -88.0, -30.0, 30.0, 88.0, 200.0, 3e38])
def test_silu_far_gates(cuda, gate):
    g = gen(7)
    x = randn(g, 3, 500)
    x[1] = gate
    x[2, ::2] = gate
    u = randn(g, 3, 500) * (0.1 if abs(gate) > 1e30 else 1)
    check(mlb.CudaSiluMulInt8DeviceInput(x, u), ref.to_codes(ref.silu_mul(x, u)))


@pytest.mark.parametrize("dtype", TYPES)
def test_values_next_to_borders(cuda, dtype):
    """Rows whose values lie within rounding errors of the codes' borders."""
    t = getattr(torch, dtype)
    g = gen(11)
    n = 8192
    w = 1 + 0.3 * randn(g, n)
    k = torch.randint(-126, 126, (16, n), device="cuda", generator=g)
    x = ((k + 0.5) / 127.0 / w).to(t)
    x[:, 17] = 1.0 / w[17]
    for i in range(4):  # a step of fp32 to either side
        x[4 * i:4 * i + 4] = torch.nextafter(x, torch.full_like(x, math.inf if i % 2 else -math.inf))[4 * i:4 * i + 4]
    check(mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5), ref.norm_codes(x, w, 1e-5), 45 * U)
    y = ((k + 0.5) / 127.0).to(t)
    y[:, 5] = 1.0
    check(mlb.CudaInt8QuantizeDeviceInput(y), ref.to_codes(y.double()))
    gate = randn(g, 16, n).abs() + 0.5
    up = (k + 0.5) / 127.0 / ref.silu_mul(gate, torch.ones_like(gate)).float()
    gate, up = gate.to(t), up.to(t)
    check(mlb.CudaSiluMulInt8DeviceInput(gate, up), ref.to_codes(ref.silu_mul(gate, up)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,pad,shift", [(512, 8, 0), (512, 3, 0), (512, 8, 1), (777, 0, 5)])
def test_strides_alignments_and_neighbours(cuda, n, pad, shift, dtype):
    """Rows inside a larger buffer; what lies around them stays as it was."""
    t = getattr(torch, dtype)
    g = gen(n + pad)
    rows = 9

    def inside():
        flat = randn(g, rows * (n + pad) + shift + 7).to(t)
        return flat, flat[shift:shift + rows * (n + pad)].view(rows, n + pad)[:, :n]

    (_, x), (_, r), (flat, out) = inside(), inside(), inside()
    w = 1 + 0.1 * randn(g, n + 1)[1:].contiguous()
    h = (x.float() + r.float()).to(t)
    keep = flat.clone()
    got = mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=r, sum_out=out)
    assert got[2] is out and torch.equal(out, h)
    check(got, ref.norm_codes(h, w, 1e-5), 45 * U)
    out.copy_(keep[shift:shift + rows * (n + pad)].view(rows, n + pad)[:, :n])
    assert torch.equal(flat, keep)
    check(mlb.CudaInt8QuantizeDeviceInput(x), ref.to_codes(x.double()))
    check(mlb.CudaSiluMulInt8DeviceInput(x, r), ref.to_codes(ref.silu_mul(x, r)))
    # columns of a transposed matrix are copied
    xt = randn(g, n, rows).to(t).t()
    check(mlb.CudaInt8QuantizeDeviceInput(xt), ref.to_codes(xt.double()))
    for into in (x, r):  # in place
        x1, r1 = x.clone(), r.clone()
        where = x1 if into is x else r1
        got = mlb.CudaRmsNormInt8DeviceWeight(x1, w, 1e-5, residual=r1, sum_out=where)
        assert torch.equal(where, h)
        check(got, ref.norm_codes(h, w, 1e-5), 45 * U)


@pytest.mark.parametrize("rows,n", [(3, 1000), (1500, 4096), (700, 777), (2, 40000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_many_equal_maxima(cuda, dtype, rows, n):
    """Clipped rows, constant rows and rows of two magnitudes among ordinary ones."""
    t = getattr(torch, dtype)
    g = gen(rows + n)
    x = randn(g, rows, n)
    x[::3] = x[::3].clamp(-1.25, 1.25)
    x[1::5] = -0.7
    x[2::7] = torch.where(x[2::7] > 0, 3.0, -1.5)
    x = x.to(t)
    w = torch.ones(n, device="cuda")
    check(mlb.CudaInt8QuantizeDeviceInput(x), ref.to_codes(x.double()))
    check(mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5), ref.norm_codes(x, w, 1e-5), 45 * U)
    w = 1 + 0.2 * randn(g, n)
    r = torch.zeros_like(x)
    check(mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=r), ref.norm_codes(x, w, 1e-5), 45 * U)
    u = torch.where(x > 0, 2.0, 1.0).to(t)
    check(mlb.CudaSiluMulInt8DeviceInput(x, u), ref.to_codes(ref.silu_mul(x, u)))
    check(mlb.CudaSiluMulInt8DeviceInput(u, x), ref.to_codes(ref.silu_mul(u, x)))


def test_long_rows_in_place(cuda):
    g = gen(3)
    x, r, w = randn(g, 2, 70001), randn(g, 2, 70001), 1 + 0.1 * randn(g, 70001)
    h = x + r
    got = mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=r, sum_out=x)
    assert torch.equal(x, h)
    check(got, ref.norm_codes(h, w, 1e-5), 60 * U)  # 69 terms a thread


def test_no_rows(cuda):
    x, w = torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda")
    for got in (mlb.CudaInt8QuantizeDeviceInput(x), mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5),
                mlb.CudaSiluMulInt8DeviceInput(x, x)):
        assert got[0].shape == (0, 64) and got[1].shape == (0,)
        assert mlb.CudaInt8DequantizeDeviceInput(*got).shape == (0, 64)
    assert len(mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=x)) == 3


def test_one_row_as_a_vector(cuda):
    g = gen(5)
    x, w = randn(g, 4096), torch.ones(4096, device="cuda")
    check(mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5), ref.norm_codes(x[None], w, 1e-5), 45 * U)
