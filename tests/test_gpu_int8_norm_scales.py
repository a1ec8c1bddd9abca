"""A norm's scales: the root's sum of squares is taken in 64 bits, so a scale is the
64-bit one rounded once, and does not depend on the rows beside it or on where they lie.

The sum has at most n / 1024 + 60 roundings of 2^-53, halved by the root: below 2^-40 for
the longest row here, 2^-47 for those of other tests. Two orders of it come to the same
fp32 number unless the 64-bit one lies that close to the middle of two, one in 2^23."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import int8_ref as ref  # noqa: E402

ONCE = 2.0 ** -24 * (1 + 2.0 ** -10)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def norm(x, w, r):
    return mlb.CudaRmsNormInt8DeviceWeight(x, w, 1e-5, residual=r)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [96, 1000, 1001, 4096, 8192, 14336, 40000])
def test_rows_beside_it(cuda, n, dtype, residual):
    """The same bits alone, among few rows, among many, and in rows that start anywhere."""
    t, g = getattr(torch, dtype), torch.Generator(device="cuda").manual_seed(n)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    many = 5 * sms
    x, w = randn(g, many, n).to(t), 1 + 0.3 * randn(g, n)
    r = (randn(g, many, n) * 2).to(t) if residual else None
    whole = norm(x, w, r)
    want = ref.norm_codes(x if r is None else whole[2], w, 1e-5)
    assert torch.equal(whole[0], want[0])
    assert ((whole[1].double() - want[1]).abs() <= want[1] * ONCE).all()
    for rows in (1, 2, sms, 2 * sms, 2 * sms + 1):
        part = norm(x[:rows], w, None if r is None else r[:rows])
        assert torch.equal(part[0], whole[0][:rows])
        assert torch.equal(part[1], whole[1][:rows]), rows
    apart = torch.empty(many, n + 3, device="cuda", dtype=t)[:, 1:n + 1]
    apart.copy_(x)
    part = norm(apart, w, r)
    assert torch.equal(part[0], whole[0]) and torch.equal(part[1], whole[1])


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [8192, 65536, 262152, (1 << 23) + 5])
def test_long_rows(cuda, n, dtype, residual):
    """Rows of equal squares, whose running sum rounds the same way at each step."""
    t = getattr(torch, dtype)
    x = torch.full((2, n), 1.1, device="cuda").to(t)
    x[1] *= 1.3
    w = torch.ones(n, device="cuda")
    r = torch.zeros_like(x) if residual else None
    got, want = norm(x, w, r), ref.norm_codes(x, w, 1e-5)
    assert torch.equal(got[0], want[0])
    assert ((got[1].double() - want[1]).abs() <= want[1] * ONCE).all()


@pytest.mark.parametrize("size", [1e-25, 1e-19, 1e-12, 1e12, 1e19, 1e25])
@pytest.mark.parametrize("n", [1000, 1001, 40000, 270000])
def test_squares_that_fp32_does_not_hold(cuda, n, size):
    g = torch.Generator(device="cuda").manual_seed(n)
    x, w = randn(g, 3, n) * size, 1 + 0.3 * randn(g, n)
    got, want = norm(x, w, None), ref.norm_codes(x, w, 1e-5)
    assert torch.equal(got[0], want[0])
    assert ((got[1].double() - want[1]).abs() <= want[1] * ONCE + 2.0 ** -150).all()
    got = mlb.CudaRmsNormInt8DeviceWeight(x, w, 0.0)
    want = ref.norm_codes(x, w, 0.0)
    assert torch.equal(got[0], want[0])
    assert ((got[1].double() - want[1]).abs() <= want[1] * ONCE + 2.0 ** -150).all()
