"""Product of int8 codes with scales for each token and channel, against 64 bits.

The sum is exact. Rounding it to fp32, the two scales and the bias are off by 2^-24
each: three of the product (its size), one of the result; bf16 adds 2^-8 of the result.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from mini_llama_b200 import _lib  # noqa: E402
from tests import int8_ref as ref  # noqa: E402

U = 2.0 ** -24


def codes(g, rows, n, lo=-127, hi=127):
    padded = torch.full((rows, (n + 15) // 16 * 16), 99, device="cuda", dtype=torch.int8)
    padded[:, :n] = torch.randint(lo, hi + 1, (rows, n), device="cuda", generator=g,
                                  dtype=torch.int8)
    return padded[:, :n]


def operands(rows, k, n, bias, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + k + n)
    x, w = codes(g, rows, k), codes(g, n, k)
    sx = torch.rand(rows, device="cuda", generator=g) + 0.01
    sw = torch.rand(n, device="cuda", generator=g) * 1e-3
    b = torch.randn(n, device="cuda", generator=g) if bias else None
    return x, sx, w, sw, b


def check(y, x, sx, w, sw, b=None):
    want, size = ref.linear(x, sx, w, sw, b)
    tol = 3 * U * size + U * want.abs()
    if y.dtype is torch.bfloat16:
        tol = tol * (1 + 2.0 ** -7) + 2.0 ** -8 * want.abs()
    err = (y.double() - want).abs()
    assert (err <= tol * (1 + 2.0 ** -20)).all(), (err / tol).max()


SHAPES = [(1, 1, 1), (1, 16, 8), (3, 17, 5), (1, 128, 128), (2, 129, 129), (16, 4096, 4096),
          (17, 4096, 130), (1, 29568, 1000), (8, 14336, 257), (32, 8192, 10240), (33, 1000, 64),
          (64, 288, 1536), (65, 640, 300), (100, 2048, 2048), (129, 1000, 257), (255, 96, 96),
          (256, 4096, 512), (257, 4096, 512), (300, 777, 999), (511, 1536, 768), (777, 288, 1536),
          (1000, 5000, 1030), (2048, 512, 4096), (1, 64, 28672), (513, 127, 131)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_linear(cuda, rows, k, n, dtype):
    for bias in (False, True):
        ops = operands(rows, k, n, bias)
        y = mlb.CudaInt8LinearDeviceInput(*ops, out_dtype=getattr(torch, dtype))
        assert y.shape == (rows, n) and y.dtype is getattr(torch, dtype)
        check(y, *ops)
        again = mlb.CudaInt8LinearDeviceInput(*ops, out_dtype=getattr(torch, dtype))
        assert torch.equal(y, again)
    assert mlb.int8_linear_status() == (0, 0)


@pytest.mark.parametrize("rows", [1, 20, 150, 600])
def test_largest_sums(cuda, rows):
    """131071 products of -128 by -128, 31 bits of sum; next to rows of both signs."""
    k, n = 131071, 140
    x = torch.full((rows, 131072), -128, device="cuda", dtype=torch.int8)[:, :k]
    w = torch.full((n, 131072), -128, device="cuda", dtype=torch.int8)[:, :k]
    w[::3] = 127
    w[1::7, ::2] = 127
    sx, sw = torch.ones(rows, device="cuda"), torch.ones(n, device="cuda")
    check(mlb.CudaInt8LinearDeviceInput(x, sx, w, sw), x, sx, w, sw)


@pytest.mark.parametrize("rows,k,n", [(1, 4096, 4096), (40, 1000, 999), (700, 512, 640)])
def test_rows_do_not_depend_on_each_other(cuda, rows, k, n):
    """A row alone gives the bits that it gives among others; a NaN scale makes its own
    row NaN, a channel's its own column."""
    x, sx, w, sw, b = operands(rows, k, n, True)
    y = mlb.CudaInt8LinearDeviceInput(x, sx, w, sw, b)
    for i in {0, rows // 2, rows - 1}:
        assert torch.equal(mlb.CudaInt8LinearDeviceInput(x[i:i + 1], sx[i:i + 1], w, sw, b)[0], y[i])
    sx2, sw2 = sx.clone(), sw.clone()
    sx2[rows // 2], sw2[3] = math.nan, math.nan
    z = mlb.CudaInt8LinearDeviceInput(x, sx2, w, sw2, b)
    bad = torch.zeros_like(z, dtype=torch.bool)
    bad[rows // 2], bad[:, 3] = True, True
    assert torch.isnan(z[bad]).all() and torch.equal(z[~bad], y[~bad])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,k,n,pad,shift", [(3, 100, 130, 5, 1), (70, 256, 200, 1, 0),
                                                (300, 512, 384, 8, 0), (513, 128, 250, 6, 2)])
def test_outputs_inside_a_buffer(cuda, rows, k, n, pad, shift, dtype):
    t = getattr(torch, dtype)
    ops = operands(rows, k, n, True)
    flat = torch.full((rows * (n + pad) + shift + 64,), 7.0, device="cuda", dtype=t)
    out = flat[shift:shift + rows * (n + pad)].view(rows, n + pad)[:, :n]
    assert mlb.CudaInt8LinearDeviceInput(*ops, out=out) is out
    check(out, *ops)
    out.fill_(7.0)
    assert (flat == 7.0).all()


def test_codes_of_other_layouts_are_copied(cuda):
    x, sx, w, sw, b = operands(5, 100, 60, False)
    want = mlb.CudaInt8LinearDeviceInput(x, sx, w, sw)
    xc, wt = x.contiguous(), w.t().contiguous().t()
    assert xc.stride(0) == 100
    assert torch.equal(mlb.CudaInt8LinearDeviceInput(xc, sx, wt, sw), want)
    wide = torch.zeros(61, 160, device="cuda", dtype=torch.int8)
    wide[1:, 16:116] = w
    assert torch.equal(mlb.CudaInt8LinearDeviceInput(x, sx, wide[1:, 16:116], sw), want)


def test_no_rows(cuda):
    x, sx, w, sw, b = operands(1, 64, 32, True)
    assert mlb.CudaInt8LinearDeviceInput(x[:0], sx[:0], w, sw, b).shape == (0, 32)


@pytest.mark.parametrize("rows", [1, 40, 200, 1000])
def test_waits_that_run_out(cuda, rows):
    code, where, nan = mlb.int8_linear_wait_selftest(rows, 1.0)
    assert code == mlb.ERR_TIMEOUT and 1101 <= where < 1120 and nan == rows
    assert mlb.int8_linear_status() == (0, 0)
    ops = operands(rows, 2048, 256, False)
    check(mlb.CudaInt8LinearDeviceInput(*ops), *ops)


def test_streams_and_graphs(cuda):
    """Two products at once on two streams, and a captured one replayed with new codes."""
    a, b = operands(1, 4096, 4096, True, 1), operands(600, 1024, 1024, True, 2)
    want = mlb.CudaInt8LinearDeviceInput(*a), mlb.CudaInt8LinearDeviceInput(*b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        got.append((mlb.CudaInt8LinearDeviceInput(*a, stream=s1.cuda_stream),
                    mlb.CudaInt8LinearDeviceInput(*b, stream=s2.cuda_stream)))
    torch.cuda.synchronize()
    for u, v in got:
        assert torch.equal(u, want[0]) and torch.equal(v, want[1])
    out = torch.empty_like(want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mlb.CudaInt8LinearDeviceInput(*a, out=out)
    other = operands(1, 4096, 4096, True, 9)
    for t, u in zip(a, other):
        t.copy_(u)
    graph.replay()
    torch.cuda.synchronize()
    check(out, *other)


@pytest.mark.parametrize("n,k", [(4096, 1024), (513, 300), (4096, 4096)])
def test_weights_that_the_kernel_before_writes(n, k):
    """Weights are asked for while the kernel before runs: one that makes them, over and
    over in the same place, is waited for all the same, in a graph too."""
    g = torch.Generator(device="cuda").manual_seed(n + k)
    many = torch.randn(6, n, k, device="cuda", generator=g)
    x, xs = mlb.CudaInt8QuantizeDeviceInput(torch.randn(3, k, device="cuda", generator=g))
    width = (k + 15) // 16 * 16
    place, scales = torch.empty(n, width, dtype=torch.int8, device="cuda"), None
    w = place[:, :k]
    want = []
    for v in many:
        codes, scales = mlb.CudaInt8QuantizeDeviceInput(v)
        want.append(mlb.CudaInt8LinearDeviceInput(x, xs, codes.clone(), scales.clone()))
    scales = torch.empty(n, device="cuda")
    lib = _lib.lib()

    def chain():
        out = []
        for v in many:
            assert lib.mlb_int8_quantize(0, v.data_ptr(), k, n, k, w.data_ptr(), width,
                                         scales.data_ptr(), 0,
                                         torch.cuda.current_stream().cuda_stream) == 0
            out.append(mlb.CudaInt8LinearDeviceInput(x, xs, w, scales))
        return out

    for made, right in zip(chain(), want):
        assert torch.equal(made, right)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    for made, right in zip(out, want):
        assert torch.equal(made, right)
