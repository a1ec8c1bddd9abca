"""A transformer layer in int8, as a serving loop runs it: norm, query-key-value product,
rotation, paged cache and attention, output product, residual and norm, gate-up product,
SiLU product, down product. Every step is checked against 64 bits on the inputs that the
step before has left, so that its own error bound holds.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import int8_ref as ref  # noqa: E402

U = 2.0 ** -24
DIM, HIDDEN, HEADS, KV, HD, ROT, PAGE, EPS = 512, 1376, 8, 2, 64, 32, 16, 1e-5


def ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


class Layer:
    def __init__(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(n, k):
            return mlb.CudaInt8QuantizeDeviceInput(
                torch.randn(n, k, device="cuda", generator=g) * k ** -0.5)

        self.qkv, self.wo = matrix((HEADS + 2 * KV) * HD, DIM), matrix(DIM, HEADS * HD)
        self.gate_up, self.down = matrix(2 * HIDDEN, DIM), matrix(DIM, HIDDEN)
        self.bias = torch.randn((HEADS + 2 * KV) * HD, device="cuda", generator=g) * 0.1
        self.norms = [1 + 0.1 * torch.randn(DIM, device="cuda", generator=g) for _ in range(2)]
        self.table = mlb.RopeTable(ROT, 500000.0, mlb.ROPE_SCALING_LLAMA3, 8.0, 8192)
        self.cache = mlb.CudaPagedKvCache(1, 40, PAGE, KV, HD)

    def run(self, x, delta, pos, offsets, lens, pages):
        """The residual stream x and the last layer's delta; everything on the way."""
        r, t = {}, x.dtype
        r["a"] = mlb.CudaRmsNormInt8DeviceWeight(x, self.norms[0], EPS, residual=delta)
        r["qkv"] = mlb.CudaInt8LinearDeviceInput(*r["a"][:2], *self.qkv, bias=self.bias, out_dtype=t)
        rows = x.shape[0]
        q, k, v = (p.view(rows, -1, HD) for p in
                   r["qkv"].split([HEADS * HD, KV * HD, KV * HD], 1))
        r["q"], r["k"] = mlb.CudaRopeRowsDeviceInput(q, k, pos, self.table)
        self.cache.AppendDevice(0, r["k"], v, offsets, lens, pages, rope_type=mlb.ROPE_NONE)
        r["att"] = mlb.CudaPagedAttentionDeviceInput(r["q"], self.cache, 0, offsets, lens, pages,
                                                     HEADS, KV, HD)
        r["att8"] = mlb.CudaInt8QuantizeDeviceInput(r["att"].view(rows, -1))
        r["o"] = mlb.CudaInt8LinearDeviceInput(*r["att8"], *self.wo, out_dtype=t)
        r["b"] = mlb.CudaRmsNormInt8DeviceWeight(r["a"][2], self.norms[1], EPS, residual=r["o"])
        r["gu"] = mlb.CudaInt8LinearDeviceInput(*r["b"][:2], *self.gate_up, out_dtype=t)
        r["s"] = mlb.CudaSiluMulInt8DeviceInput(*r["gu"].split(HIDDEN, 1))
        r["out"] = mlb.CudaInt8LinearDeviceInput(*r["s"], *self.down, out_dtype=t)
        return r

    def check(self, r, x, delta, pos, lens, new):
        t = x.dtype

        def rounds(y, want, tol):
            if t is torch.bfloat16:
                tol = tol * (1 + 2.0 ** -7) + 2.0 ** -8 * want.abs()
            assert ((y.double() - want).abs() <= tol).all()

        def product(y, x8, w8, bias=None):
            want, size = ref.linear(*x8, *w8, bias)
            rounds(y, want, 3 * U * size + U * want.abs())

        def codes(got, want, tol):
            assert torch.equal(got[0], want[0])
            assert ((got[1].double() - want[1]).abs() <= tol * want[1]).all()

        h = (x.float() + delta.float()).to(t)
        assert torch.equal(r["a"][2], h)
        codes(r["a"], ref.norm_codes(h, self.norms[0], EPS), 45 * U)
        product(r["qkv"], r["a"][:2], self.qkv, self.bias)
        q, k, _ = (p.view(x.shape[0], -1, HD) for p in
                   r["qkv"].split([HEADS * HD, KV * HD, KV * HD], 1))
        f = self.table.frequencies.cpu()
        for got, src in ((r["q"], q), (r["k"], k)):
            want = ref.rope(src, pos, f, 1.0, False)
            # |a| + |b| of a pair is at most sqrt 2 of its length, which turning keeps
            pair = src.double().view(*src.shape[:2], -1, 2).norm(dim=-1).repeat_interleave(2, -1)
            rounds(got, want, 12 * U * 1.4143 * pair)
        codes(r["att8"], ref.to_codes(r["att"].view(x.shape[0], -1).double()), U)
        product(r["o"], r["att8"], self.wo)
        h = (h.float() + r["o"].float()).to(t)
        assert torch.equal(r["b"][2], h)
        codes(r["b"], ref.norm_codes(h, self.norms[1], EPS), 45 * U)
        product(r["gu"], r["b"][:2], self.gate_up)
        codes(r["s"], ref.to_codes(ref.silu_mul(*r["gu"].split(HIDDEN, 1))), U)
        product(r["out"], r["s"], self.down)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_layer(cuda, dtype):
    """Two prompts, then decode steps of both replayed from one graph on a stream of
    its own, each step's positions and lengths new."""
    t = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    layer = Layer(5)
    pages = ints([list(range(0, 20)), list(range(20, 40))])
    new = [150, 33]

    def inputs(rows):
        return [(torch.randn(rows, DIM, device="cuda", generator=g) * s).to(t) for s in (1.0, 0.3)]

    x, delta = inputs(sum(new))
    pos = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in new])
    lens = ints(new)
    r = layer.run(x, delta, pos, ints([0, 150, 183]), lens, pages)
    layer.check(r, x, delta, pos, new, new)

    x, delta = inputs(2)
    pos, offsets = lens.clone(), ints([0, 1, 2])
    lens = lens + 1
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer.run(x, delta, pos, offsets, lens, pages)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            r = layer.run(x, delta, pos, offsets, lens, pages)
        for _ in range(3):
            for old, fresh in zip((x, delta), inputs(2)):
                old.copy_(fresh)
            graph.replay()
            stream.synchronize()
            layer.check(r, x, delta, pos, lens.tolist(), [1, 1])
            eager = layer.run(x, delta, pos, offsets, lens, pages)
            assert torch.equal(eager["out"], r["out"])
            pos += 1
            lens += 1
    assert mlb.int8_linear_status() == (0, 0) and mlb.paged_attention_status() == (0, 0)
