"""Whole numbers and sizes past 32 bits are refused: the C ABI takes ints, and the lower
bits alone would name another type, another scaling or a smaller call."""
import pytest

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402

FAR = [1 << 32, (1 << 32) + 1, -(1 << 32), 1 << 31, 1 << 70]


@pytest.mark.parametrize("far", FAR)
def test_numbers_are_refused_before_the_device(far):
    for call in (lambda: mlb.RopeTable(64, scaling=far), lambda: mlb.RopeTable(far + 64),
                 lambda: mlb.int8_linear_wait_selftest(rows=far + 8),
                 lambda: mlb.int8_linear_wait_selftest(device_id=far),
                 lambda: mlb.int8_linear_status(far)):
        with pytest.raises(mlb.MlbError, match="out of range"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("far", FAR)
def test_rope_types(cuda, far):
    q, pos = torch.randn(2, 1, 32, device="cuda"), torch.zeros(2, device="cuda", dtype=torch.int32)
    table = mlb.RopeTable(32)
    assert mlb._load_calls().rope_rows(q, q, pos, table.frequencies, 1.0, far) is None
    assert mlb._load_calls().int8_dequantize(*mlb.CudaInt8QuantizeDeviceInput(q[:, 0]), far) is None
    for k, out in ((q, None), (None, None), (q.clone(), torch.empty_like(q))):
        with pytest.raises(mlb.MlbError, match="rope type"):
            mlb.CudaRopeRowsDeviceInput(q, k, pos, table, rope_type=far, q_out=out)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(1, (1 << 32) + 64), (2, (1 << 32) + 64), ((1 << 32) + 2, 64)])
def test_sizes(cuda, rows, n):
    """Nothing is copied or launched for them (the rows take no memory here)."""
    x = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16).expand(rows, n)
    c, s = x[:1, :1].to(torch.int8).expand(rows, n), x[:1, 0].float().expand(rows)
    w = s[:1].expand(n)
    b, bs = mlb.CudaInt8QuantizeDeviceInput(torch.ones(8, 64, device="cuda"))
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for call in (lambda: mlb.CudaInt8QuantizeDeviceInput(x),
                 lambda: mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5),
                 lambda: mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=x),
                 lambda: mlb.CudaSiluMulInt8DeviceInput(x, x),
                 lambda: mlb.CudaInt8DequantizeDeviceInput(c, s),
                 lambda: mlb.CudaInt8LinearDeviceInput(c, s, b, bs),
                 lambda: mlb.CudaInt8LinearDeviceInput(b, bs, c, s)):
        with pytest.raises(mlb.MlbError, match="out of range"):
            call()
    assert torch.cuda.max_memory_allocated() - before < 1 << 20


@pytest.mark.gpu
def test_rotated_sizes(cuda):
    one = torch.zeros(1, 1, 1, device="cuda", dtype=torch.bfloat16)
    pos, table = torch.zeros(1, device="cuda", dtype=torch.int32), mlb.RopeTable(32)
    for shape in ((1, (1 << 32) + 1, 32), (1, 1, (1 << 32) + 32)):
        with pytest.raises(mlb.MlbError, match="out of range"):
            mlb.CudaRopeRowsDeviceInput(one.expand(shape), None, pos, table)
