"""Rows as int8 codes that several CTAs share, or that one passes over twice.

Codes are the 64-bit form's, every one. Scales: A / 127 (times the root) rounded once; the
root's sum of squares is fp32: up to 32 terms one after another in a thread (n / 1024 of
rows past 262144 elements), a tree of at most 42 more steps and 8 CTAs' sums, each off by
2^-24, half of which the square root passes on, and 4 more roundings.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import int8_ref as ref  # noqa: E402

U = 2.0 ** -24
TYPES = ["float32", "bfloat16"]
# rows of one CTA's registers and a little more, of two to eight CTAs', of more; few rows that
# share what one CTA could hold, to either side of where they begin to
SHAPES = [(1, 8192), (1, 8200), (2, 16385), (16, 29568), (37, 16392), (74, 14336), (75, 14336),
          (148, 20000), (1, 32768), (1, 32769), (200, 33000), (3, 65536), (2, 65537), (2, 131080),
          (1, 262144), (2, 262145), (3, 300008)]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def norm_tol(n):
    return ((32 if n <= 262144 else n / 1024 + 1) + 50) / 2 * U + 4 * U


def check(got, want, tol=U):
    assert torch.equal(got[0], want[0]), (got[0] != want[0]).sum()
    err = (got[1].double() - want[1]).abs()
    assert (err <= want[1] * tol + 2.0 ** -150).all(), (err / want[1]).max() / U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_every_kind(cuda, rows, n, dtype):
    t, g = getattr(torch, dtype), gen(rows + n)
    x, y, w = randn(g, rows, n).to(t), (randn(g, rows, n) * 2).to(t), 1 + 0.3 * randn(g, n)
    check(mlb.CudaInt8QuantizeDeviceInput(x), ref.to_codes(x.double()))
    check(mlb.CudaSiluMulInt8DeviceInput(y, x), ref.to_codes(ref.silu_mul(y, x)))
    check(mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5), ref.norm_codes(x, w, 1e-5), norm_tol(n))
    h = (x.float() + y.float()).to(t)
    want = ref.norm_codes(h, w, 1e-5)
    for place in (None, x, y):
        a, b = (x.clone(), y.clone())
        out = None if place is None else a if place is x else b
        got = mlb.CudaRmsNormInt8DeviceWeight(a, w, 1e-5, residual=b, sum_out=out)
        assert torch.equal(got[2], h)
        check(got, want, norm_tol(n))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [29568, 33001, 65536, 270000])
def test_rows_of_any_kind(cuda, n, dtype):
    """Rows that fp32 cannot hold the bounds for, and NaN or an infinity in one part of a
    row alone."""
    t = getattr(torch, dtype)
    x = randn(gen(n), 10, n)
    x[0] = 0.0
    x[1] = 0.0
    x[1, n - 2] = -5.0
    x[2] *= 1e-33
    x[3] *= 1e-39
    x[4] = x[4].clamp(-3, 3) * 1e38
    x[5, 3] = math.nan
    x[6, n - 1] = math.inf
    x[7, n // 2] = -math.inf
    x[8] *= 1e18
    x = x.to(t)
    ok = torch.tensor([i not in (5, 6, 7) for i in range(10)], device="cuda")
    w, none = 1 + 0.2 * randn(gen(n + 1), n), torch.zeros_like(x)
    one = torch.ones_like(x)
    far = one.clone()
    far[:, n // 3] = -90.0  # a gate below what fp32's form takes, in one part
    for got, want, tol in (
            (mlb.CudaInt8QuantizeDeviceInput(x), ref.to_codes(x.double()), U),
            (mlb.CudaSiluMulInt8DeviceInput(one, x), ref.to_codes(ref.silu_mul(one, x)), U),
            (mlb.CudaSiluMulInt8DeviceInput(far, x), ref.to_codes(ref.silu_mul(far, x)), U),
            (mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5), ref.norm_codes(x, w, 1e-5), norm_tol(n)),
            (mlb.CudaRmsNormInt8DeviceWeight(x.clone(), w, 1e-5, residual=none.clone()),
             ref.norm_codes(x, w, 1e-5), norm_tol(n))):
        check((got[0][ok], got[1][ok]), (want[0][ok], want[1][ok]), tol)
        assert got[1][~ok].isnan().all()
    a = x.clone()
    in_place = mlb.CudaRmsNormInt8DeviceWeight(a, w, 1e-5, residual=none, sum_out=a)
    apart = mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=none)
    assert torch.equal(in_place[0][ok], apart[0][ok]) and torch.equal(in_place[1][ok], apart[1][ok])


@pytest.mark.parametrize("rows,n", [(16, 29568), (2, 65536), (160, 40000)])
def test_values_next_to_borders(cuda, rows, n):
    """Values within rounding errors of the codes' borders, and many in each CTA's part that
    fp32 cannot tell from the maximum."""
    g = gen(n)
    k = torch.randint(-126, 126, (rows, n), device="cuda", generator=g)
    k[:, ::1000] = 125
    gate = randn(g, rows, n).abs() + 0.5
    up = (k + 0.5) / 127.0 / ref.silu_mul(gate, torch.ones_like(gate)).float()
    check(mlb.CudaSiluMulInt8DeviceInput(gate, up), ref.to_codes(ref.silu_mul(gate, up)))
    w = 1 + 0.3 * randn(g, n)
    x = ((k + 0.5) / 127.0 / w).float()
    check(mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5), ref.norm_codes(x, w, 1e-5), norm_tol(n))


def test_again_and_in_a_graph(cuda):
    """The same bits every time: eager, among other calls, captured and replayed."""
    g = gen(5)
    x, y, w = randn(g, 3, 65536), randn(g, 3, 65536), randn(g, 65536)
    gate, up = randn(g, 16, 29568), randn(g, 16, 29568)

    def calls():
        return [*mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=y),
                *mlb.CudaSiluMulInt8DeviceInput(gate, up), *mlb.CudaInt8QuantizeDeviceInput(x)]

    want = calls()
    for _ in range(20):
        for a, b in zip(calls(), want):
            assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = calls()
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(made, want):
        assert torch.equal(a, b)
