"""Views that torch reads negated (imaginary parts of conjugates): inputs are taken as the
values that torch shows, vectors and outputs that cannot be are refused."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402


def negated(*shape):
    z = torch.randn(*shape, dtype=torch.complex64, device="cuda")
    v = z.conj().imag
    assert v.is_neg()
    return v


def same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,n", [(4, 1), (1, 1), (3, 40)])
def test_rows(cuda, rows, n):
    x, y = negated(rows, n), negated(rows, n)
    a, b = x.clone(), y.clone()
    assert not a.is_neg()
    w = torch.rand(n, device="cuda")
    same(mlb.CudaInt8QuantizeDeviceInput(x), mlb.CudaInt8QuantizeDeviceInput(a))
    same(mlb.CudaSiluMulInt8DeviceInput(x, y), mlb.CudaSiluMulInt8DeviceInput(a, b))
    for out in (None, torch.empty_like(a)):
        same(mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=y, sum_out=out),
             mlb.CudaRmsNormInt8DeviceWeight(a, w, 1e-5, residual=b))


def test_rotation(cuda):
    q, pos = negated(3, 1, 2), torch.arange(3, device="cuda", dtype=torch.int32)
    table = mlb.RopeTable(2)
    want = mlb.CudaRopeRowsDeviceInput(q.clone(), q.clone(), pos, table)
    same(mlb.CudaRopeRowsDeviceInput(q, q, pos, table), want)
    flat = torch._neg_view(q.clone().neg())
    assert flat.is_contiguous() and torch.equal(flat, q)
    same(mlb.CudaRopeRowsDeviceInput(flat, flat, pos, table), want)


def test_vectors_and_outputs_are_refused(cuda):
    x, one = torch.randn(1, 1, device="cuda"), negated(1)
    c, s = mlb.CudaInt8QuantizeDeviceInput(x)
    q, pos = x.view(1, 1, 1).expand(1, 1, 2), torch.zeros(1, device="cuda", dtype=torch.int32)
    table = mlb.RopeTable(2)
    for call in (lambda: mlb.CudaRmsNormInt8DeviceWeight(x, one, 1e-5),
                 lambda: mlb.CudaRmsNormInt8DeviceWeight(x, s, 1e-5, residual=x, sum_out=one[None]),
                 lambda: mlb.CudaInt8DequantizeDeviceInput(c, one),
                 lambda: mlb.CudaInt8LinearDeviceInput(c, one, c, s),
                 lambda: mlb.CudaInt8LinearDeviceInput(c, s, c, one),
                 lambda: mlb.CudaInt8LinearDeviceInput(c, s, c, s, bias=one),
                 lambda: mlb.CudaInt8LinearDeviceInput(c, s, c, s, out=one[None]),
                 lambda: mlb.CudaRopeRowsDeviceInput(q, None, pos, table, q_out=torch._neg_view(
                     torch.zeros(1, 1, 2, device="cuda")))):
        with pytest.raises(mlb.MlbError, match="negated view"):
            call()
