"""The int8 layer's calls where a program could trip over them: offsets past 32 bits,
streams beside one another, graphs replayed on new data, tensors of wrong kinds."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import int8_ref as ref  # noqa: E402


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes(g, rows, n):
    width = (n + 15) // 16 * 16
    return torch.randint(-127, 128, (rows, width), device="cuda", generator=g,
                         dtype=torch.int8)[:, :n]


def test_rows_past_32_bits(cuda):
    """2.3e9 elements: the last rows come out as they do alone."""
    g = gen(1)
    rows, n, last = 70016, 32768, 5
    x = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
    x[:] = torch.randn(1, n, device="cuda", generator=g).to(x.dtype)
    x[-last:] = torch.randn(last, n, device="cuda", generator=g).to(x.dtype)
    w = 1 + 0.2 * torch.randn(n, device="cuda", generator=g)
    assert x.numel() > 2 ** 31
    r = x.clone()
    alone = mlb.CudaRmsNormInt8DeviceWeight(x[-last:].clone(), w, 1e-5, residual=r[-last:].clone())
    got = mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=r, sum_out=x)
    for a, b in zip(alone, got):
        assert torch.equal(a, b[-last:])
    del x
    back = mlb.CudaInt8DequantizeDeviceInput(got[0], got[1], out_dtype=torch.bfloat16)
    assert torch.equal(back[-last:], mlb.CudaInt8DequantizeDeviceInput(
        alone[0], alone[1], out_dtype=torch.bfloat16))
    del back
    for call in (lambda t: mlb.CudaInt8QuantizeDeviceInput(t),
                 lambda t: mlb.CudaSiluMulInt8DeviceInput(t, t)):
        whole, part = call(r), call(r[-last:].clone())
        assert torch.equal(whole[0][-last:], part[0]) and torch.equal(whole[1][-last:], part[1])
    # the same codes as a product's rows, and as its weights
    other = codes(g, 64, n)
    so = torch.rand(64, device="cuda", generator=g)
    a = mlb.CudaInt8LinearDeviceInput(got[0], got[1], other, so)
    assert torch.equal(a[-last:], mlb.CudaInt8LinearDeviceInput(alone[0], alone[1], other, so))
    b = mlb.CudaInt8LinearDeviceInput(other, so, got[0], got[1])
    assert torch.equal(b[:, -last:], mlb.CudaInt8LinearDeviceInput(other, so, alone[0], alone[1]))


@pytest.mark.parametrize("rows,n", [(150016, 16384), (60, 2 ** 25 + 2 ** 24)])
def test_products_past_32_bits(cuda, rows, n):
    """2.5e9 and 3.0e9 results, of the form for many tokens and of that for few."""
    g = gen(2)
    x, w = codes(g, rows, 32), codes(g, n, 32)
    sx = torch.rand(rows, device="cuda", generator=g)
    sw = torch.rand(n, device="cuda", generator=g)
    y = mlb.CudaInt8LinearDeviceInput(x, sx, w, sw, out_dtype=torch.bfloat16)
    assert y.numel() > 2 ** 31 and mlb.int8_linear_status() == (0, 0)
    part = mlb.CudaInt8LinearDeviceInput(x[-3:], sx[-3:], w[-2000:], sw[-2000:],
                                         out_dtype=torch.bfloat16)
    assert torch.equal(y[-3:, -2000:], part)
    part = mlb.CudaInt8LinearDeviceInput(x[:3], sx[:3], w[:2000], sw[:2000],
                                         out_dtype=torch.bfloat16)
    assert torch.equal(y[:3, :2000], part)


def test_rotation_past_32_bits(cuda):
    g = gen(3)
    rows = 140000
    x = torch.empty(rows, 128, 128, device="cuda", dtype=torch.bfloat16)
    x[:] = torch.randn(1, 128, 128, device="cuda", generator=g).to(x.dtype)
    pos = torch.arange(rows, device="cuda", dtype=torch.int32)
    tab = mlb.RopeTable(128)
    part = mlb.CudaRopeRowsDeviceInput(x[-3:].clone(), None, pos[-3:].clone(), tab)[0]
    assert x.numel() > 2 ** 31
    assert mlb.CudaRopeRowsDeviceInput(x, None, pos, tab, q_out=x)[0] is x
    assert torch.equal(x[-3:], part)


def test_streams_beside_one_another(cuda):
    """Every call on a stream of its own, many times over, gives what it gives alone."""
    g = gen(4)
    x = torch.randn(900, 2048, device="cuda", generator=g)
    w = 1 + 0.1 * torch.randn(2048, device="cuda", generator=g)
    c, s = mlb.CudaInt8QuantizeDeviceInput(x)
    wc, ws = mlb.CudaInt8QuantizeDeviceInput(torch.randn(1024, 2048, device="cuda", generator=g))
    q = torch.randn(900, 8, 128, device="cuda", generator=g)
    pos = torch.arange(900, device="cuda", dtype=torch.int32)
    tab = mlb.RopeTable(64)
    calls = [lambda st: mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=x, stream=st),
             lambda st: mlb.CudaSiluMulInt8DeviceInput(x, x, stream=st),
             lambda st: mlb.CudaInt8DequantizeDeviceInput(c, s, stream=st),
             lambda st: (mlb.CudaInt8LinearDeviceInput(c, s, wc, ws, stream=st),),
             lambda st: (mlb.CudaInt8LinearDeviceInput(c[:7], s[:7], wc, ws, stream=st),),
             lambda st: (mlb.CudaInt8LinearDeviceInput(c[:100], s[:100], wc, ws, stream=st),),
             lambda st: mlb.CudaRopeRowsDeviceInput(q, None, pos, tab, stream=st)[:1]]
    want = [call(None) for call in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[call(st.cuda_stream) for call, st in zip(calls, streams)] for _ in range(15)]
    torch.cuda.synchronize()
    for turn in got:
        for a, b in zip(turn, want):
            for u, v in zip(a, b):
                assert torch.equal(u, v)


def test_chains_of_short_kernels(cuda):
    """Each kernel starts while the one before ends: what it reads must be what that one
    wrote, from the first row to the last, over and over."""
    g = gen(5)
    x = torch.randn(33, 512, device="cuda", generator=g)
    w = torch.ones(512, device="cuda")
    wc, ws = mlb.CudaInt8QuantizeDeviceInput(torch.randn(512, 512, device="cuda", generator=g) * 0.05)

    def chain(h):
        for _ in range(25):
            c, s, h = mlb.CudaRmsNormInt8DeviceWeight(h, w, 1e-5, residual=h)
            y = mlb.CudaInt8LinearDeviceInput(c, s, wc, ws)
            h = mlb.CudaInt8DequantizeDeviceInput(*mlb.CudaSiluMulInt8DeviceInput(y, y))
        return h

    slow = x
    for _ in range(25):
        c, s, slow = mlb.CudaRmsNormInt8DeviceWeight(slow, w, 1e-5, residual=slow)
        torch.cuda.synchronize()
        y = mlb.CudaInt8LinearDeviceInput(c, s, wc, ws)
        torch.cuda.synchronize()
        c, s = mlb.CudaSiluMulInt8DeviceInput(y, y)
        torch.cuda.synchronize()
        slow = mlb.CudaInt8DequantizeDeviceInput(c, s)
        torch.cuda.synchronize()
    for _ in range(5):
        assert torch.equal(chain(x), slow)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(x)
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, slow)


def test_outputs_do_not_touch_their_neighbours(cuda):
    """Codes inside a larger buffer through the C ABI: padding and other rows stay."""
    g = gen(6)
    lib, st = mlb._lib.lib(), torch.cuda.current_stream().cuda_stream
    for rows, n, stride in ((5, 37, 64), (700, 96, 112), (3, 40001, 40064)):
        x = torch.randn(rows, n, device="cuda", generator=g)
        out = torch.full((rows + 2, stride), 55, device="cuda", dtype=torch.int8)
        s = torch.full((rows + 2,), 9.0, device="cuda")
        want = ref.to_codes(x.double())
        assert lib.mlb_int8_quantize(0, x.data_ptr(), n, rows, n, out[1:].data_ptr(), stride,
                                     s[1:].data_ptr(), 0, st) == 0
        assert torch.equal(out[1:-1, :n], want[0])
        assert (out[0] == 55).all() and (out[-1] == 55).all() and (out[1:-1, n:] == 55).all()
        assert s[0] == 9 and s[-1] == 9 and not (s[1:-1] == 9).any()


def test_wrong_tensors_are_refused(cuda):
    x = torch.randn(4, 64, device="cuda")
    c, s = mlb.CudaInt8QuantizeDeviceInput(x)
    w = torch.ones(64, device="cuda")
    err = lambda text: pytest.raises(mlb.MlbError, match=text)  # noqa: E731
    with err("expected contiguous float32 weights"):
        mlb.CudaRmsNormInt8DeviceWeight(x, w.bfloat16(), 1e-5)
    with err("expected contiguous float32 weights"):
        mlb.CudaRmsNormInt8DeviceWeight(x, w[:63], 1e-5)
    with err("weights is on cpu"):
        mlb.CudaRmsNormInt8DeviceWeight(x, w.cpu(), 1e-5)
    with err("x and residual differ in type"):
        mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=x.bfloat16())
    with err("expected residual"):
        mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=x[:3])
    with err("sum_out without a residual"):
        mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, sum_out=x)
    with err("sum_out must be shaped like x"):
        mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=x, sum_out=x[:, :63])
    with err("sum must not overlap"):
        both = torch.randn(5, 64, device="cuda")
        mlb.CudaRmsNormInt8DeviceWeight(both[:4], w, 1e-5, residual=x, sum_out=both[1:])
    with err("eps must be"):
        mlb.CudaRmsNormInt8DeviceWeight(x, w, math.nan)
    with err("at least one element"):
        mlb.CudaInt8QuantizeDeviceInput(x[:, :0])
    with err("gate and up differ in type"):
        mlb.CudaSiluMulInt8DeviceInput(x, x.bfloat16())
    with err("expected up"):
        mlb.CudaSiluMulInt8DeviceInput(x, x[:, :32])
    with err("dimension mismatch"):
        mlb.CudaInt8LinearDeviceInput(c, s, c[:, :48], s)
    with err("expected contiguous float32 w_scale"):
        mlb.CudaInt8LinearDeviceInput(c, s, c, s[:3])
    with err("w is on cpu"):
        mlb.CudaInt8LinearDeviceInput(c, s, c.cpu(), s)
    with err("expected contiguous float32 bias"):
        mlb.CudaInt8LinearDeviceInput(c, s, c, s, bias=s.bfloat16())
    with err("out must be"):
        mlb.CudaInt8LinearDeviceInput(c, s, c, s, out=torch.empty(4, 5, device="cuda"))
    q, pos, tab = x.view(4, 2, 32), torch.zeros(4, device="cuda", dtype=torch.int32), mlb.RopeTable(32)
    with err("int32 positions"):
        mlb.CudaRopeRowsDeviceInput(q, None, pos.long(), tab)
    with err("int32 positions"):
        mlb.CudaRopeRowsDeviceInput(q, None, pos[:3], tab)
    with err("neither q nor k"):
        mlb.CudaRopeRowsDeviceInput(None, None, pos, tab)
    with err("expected k"):
        mlb.CudaRopeRowsDeviceInput(q, q.bfloat16(), pos, tab)
    with err("k_out without k"):
        mlb.CudaRopeRowsDeviceInput(q, None, pos, tab, k_out=q)
    with err("q_out must be shaped like q"):
        mlb.CudaRopeRowsDeviceInput(q, None, pos, tab, q_out=q[:3])
    with err("q_out must not overlap k"):
        mlb.CudaRopeRowsDeviceInput(q.clone(), q, pos, tab, q_out=q)
    with err("rotary_dim must be even, 2 to head_dim"):
        mlb.CudaRopeRowsDeviceInput(q, None, pos, mlb.RopeTable(64))
    with err("unknown rope type"):
        mlb.CudaRopeRowsDeviceInput(q, None, pos, tab, rope_type=mlb.ROPE_NONE)
