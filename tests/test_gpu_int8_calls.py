"""The int8 layer's calls have two forms: one for plain arguments, without the interpreter,
and one in Python for the rest. Both give the same bits; each takes what it should."""
import threading
import time

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402


class Never:
    """Leaves every call to the Python forms."""

    def __getattr__(self, name):
        return lambda *args: None


class Counting:
    """Which calls the plain form took."""

    def __init__(self, calls):
        self.calls, self.taken = calls, []

    def __getattr__(self, name):
        def call(*args):
            made = getattr(self.calls, name)(*args)
            self.taken.append(made is not None)
            return made
        return call


def flat(made):
    return [made] if torch.is_tensor(made) else [t for t in made if t is not None]


def calls(rows, n, dtype):
    """(name, call, whether the plain form takes it)"""
    g = torch.Generator(device="cuda").manual_seed(rows * n)
    t = getattr(torch, dtype)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(t)

    x, r, both = randn(rows, n), randn(rows, n), randn(rows, 2 * n)
    w = torch.rand(n, device="cuda", generator=g)
    c, s = mlb.CudaInt8QuantizeDeviceInput(x)
    wc, ws = mlb.CudaInt8QuantizeDeviceInput(randn(50, n))
    b = torch.rand(50, device="cuda", generator=g)
    q, k = randn(rows, 4, 32), randn(rows, 2, 32)
    qkv = randn(rows, 8 * 32)
    pos = torch.arange(rows, device="cuda", dtype=torch.int32)
    tab = mlb.RopeTable(16)
    st = torch.cuda.Stream().cuda_stream
    torch.cuda.synchronize()
    some = rows > 0
    return [
        ("norm", lambda: mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5), some),
        ("norm, residual", lambda: mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=r), some),
        ("norm, strided", lambda: mlb.CudaRmsNormInt8DeviceWeight(both[:, n:], w, 1e-5, residual=r),
         some),
        ("norm, transposed", lambda: mlb.CudaRmsNormInt8DeviceWeight(
            x.t().contiguous().t(), w, 1e-5), some and (rows == 1 or n == 1)),
        ("norm, sum_out", lambda: mlb.CudaRmsNormInt8DeviceWeight(
            x, w, 1e-5, residual=r, sum_out=torch.empty_like(x)), None),
        ("quantize", lambda: mlb.CudaInt8QuantizeDeviceInput(x), some),
        ("quantize, stream", lambda: mlb.CudaInt8QuantizeDeviceInput(x, stream=st), some),
        ("silu", lambda: mlb.CudaSiluMulInt8DeviceInput(both[:, :n], both[:, n:]), some),
        ("back", lambda: mlb.CudaInt8DequantizeDeviceInput(c, s), some),
        ("back, bf16", lambda: mlb.CudaInt8DequantizeDeviceInput(c, s, out_dtype=torch.bfloat16),
         some),
        ("product", lambda: mlb.CudaInt8LinearDeviceInput(c, s, wc, ws), some),
        ("product, bias", lambda: mlb.CudaInt8LinearDeviceInput(c, s, wc, ws, bias=b, out_dtype=t),
         some),
        ("product, unaligned", lambda: mlb.CudaInt8LinearDeviceInput(
            c, s, torch.cat([wc[:, :1].expand(50, 5), wc], 1)[:, 5:], ws), False),
        ("product, vector", lambda: mlb.CudaInt8LinearDeviceInput(c[0], s[:1], wc, ws) if some
         else c, False if some else None),
        ("rotation", lambda: mlb.CudaRopeRowsDeviceInput(q, k, pos, tab), some),
        ("rotation, neox", lambda: mlb.CudaRopeRowsDeviceInput(q, k, pos, tab, mlb.ROPE_NEOX), some),
        ("rotation, one product's rows", lambda: mlb.CudaRopeRowsDeviceInput(
            qkv[:, :128].view(rows, 4, 32), qkv[:, 128:192].view(rows, 2, 32), pos, tab), some),
        ("rotation, queries", lambda: mlb.CudaRopeRowsDeviceInput(q, None, pos, tab), False),
    ]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,n", [(1, 64), (5, 37), (300, 96), (0, 32), (3, 1)])
def test_both_forms(cuda, rows, n, dtype, monkeypatch):
    plain = mlb._load_calls()
    for name, call, takes in calls(rows, n, dtype):
        count = Counting(plain)
        monkeypatch.setattr(mlb, "_fast", count)
        first = flat(call())
        if takes is not None:
            assert count.taken == [takes], name
        monkeypatch.setattr(mlb, "_fast", Never())
        second = flat(call())
        torch.cuda.synchronize()
        assert len(first) == len(second), name
        for u, v in zip(first, second):
            assert u.dtype is v.dtype and u.shape == v.shape and u.device == v.device, name
            assert u.stride() == v.stride() or 0 in u.shape or u.shape[0] == 1, name
            assert torch.equal(u, v), name


def test_what_the_plain_form_leaves(cuda):
    """Nothing raises in it, whatever it is given."""
    f = mlb._load_calls()
    x, w = torch.randn(2, 32, device="cuda"), torch.ones(32, device="cuda")
    c, s = mlb.CudaInt8QuantizeDeviceInput(x)
    q, pos = x.view(2, 1, 32), torch.zeros(2, device="cuda", dtype=torch.int32)
    tab = mlb.RopeTable(32).frequencies
    for args in ((), (x,), (x, w, 1e-5), (x, w, "eps", None), (x, w, 1e-5, 3), (x, w, -1.0, None),
                 (x.half(), w, 1e-5, None), (x, w[:31], 1e-5, None), (x, w.cpu(), 1e-5, None),
                 (x[0], w, 1e-5, None), (x, w, 1e-5, x.cpu()), (x, w, 1e-5, x[:1]),
                 (x.to_sparse(), w, 1e-5, None), (None, None, None, None)):
        assert f.rmsnorm_int8(*args) is None
    for args in ((c, s, c, s, None), (c, s, c, s, None, 7), (c, s, c[:, :16], s, None, 0),
                 (c, s[:1], c, s, None, 0), (c, s, c, s, s[:1], 0), (x, s, c, s, None, 0),
                 (c, s, c, s, None, "bf16"), (c.cpu(), s, c, s, None, 0), (c, s, c, s, None, None)):
        assert f.int8_linear(*args) is None
    for args in ((q, q, pos, tab, 1.0, 5), (q, q, pos.long(), tab, 1.0, 0), (q, q, pos[:1], tab, 1.0, 0),
                 (q, q.bfloat16(), pos, tab, 1.0, 0), (q, None, pos, tab, 1.0, 0),
                 (q, q[..., :16], pos, tab, 1.0, 0), (q[..., :16], q[..., :16], pos, tab, 1.0, 0),
                 (q, q, pos, tab, float("nan"), 0), (q, q, pos, tab, None, 0)):
        assert f.rope_rows(*args) is None
    assert f.int8_quantize(x[:, :0]) is None and f.int8_quantize(5) is None
    assert f.silu_mul_int8(x, x[:1]) is None and f.silu_mul_int8(x, x.bfloat16()) is None
    assert f.int8_dequantize(c, s, 2) is None and f.int8_dequantize(c, s[:1], 0) is None


def test_memory_that_is_not_there(cuda):
    """Outputs that no GPU holds: torch's own error, and the next call as ever."""
    x = torch.zeros(1, 16, device="cuda", dtype=torch.int8).expand(1 << 20, 16).contiguous()
    s = torch.zeros(1 << 20, device="cuda")
    with pytest.raises(torch.OutOfMemoryError):
        mlb.CudaInt8LinearDeviceInput(x, s, x, s)
    y = mlb.CudaInt8LinearDeviceInput(x[:4], s[:4], x[:4], s[:4])
    assert y.shape == (4, 4) and not y.any()


def test_another_thread_goes_on_while_a_call_waits_for_the_queue():
    """More launches than the device's queue takes, behind a wait of a second and a half:
    a call that waits for room there holds no interpreter lock."""
    x = torch.randn(1, 256, device="cuda")
    mlb.CudaInt8QuantizeDeviceInput(x)
    torch.cuda.synchronize()
    going, worst = True, 0.0

    def tick():
        nonlocal worst
        last = time.perf_counter()
        while going:
            time.sleep(0.001)
            now = time.perf_counter()
            worst, last = max(worst, now - last), now

    other = threading.Thread(target=tick)
    other.start()
    try:
        torch.cuda._sleep(3_000_000_000)
        for _ in range(4000):
            codes, scales = mlb.CudaInt8QuantizeDeviceInput(x)
        torch.cuda.synchronize()
    finally:
        going = False
        other.join()
    assert worst < 0.5, worst
    want, want_scales = mlb.CudaInt8QuantizeDeviceInput(x)
    assert torch.equal(codes, want) and torch.equal(scales, want_scales)
