"""SiLU(gate) * up where one factor is below fp32's normal numbers and the other large
enough to bring the product back: codes are the 64-bit form's, every one, and scales
A / 127 rounded once."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import int8_ref as ref  # noqa: E402

U = 2.0 ** -24
# one row, few, more than there are SMs to hold at once; unaligned; shared by a cluster; passed
# over twice
SHAPES = [(1, 4), (3, 96), (2, 101), (1, 29568), (2, 40000), (1500, 1024), (700, 777), (1, 270000)]


def check(gate, up):
    codes, scales = mlb.CudaSiluMulInt8DeviceInput(gate, up)
    want, want_scales = ref.to_codes(ref.silu_mul(gate, up))
    assert torch.equal(codes, want), ((codes != want).sum(), codes.numel())
    err = (scales.double() - want_scales).abs()
    assert (err <= want_scales * U + 2.0 ** -150).all()


def test_four_subnormal_gates(cuda):
    gate = torch.tensor([[4.0, 3.0, 1.0, 5.0]], dtype=torch.float64, device="cuda") * 2.0 ** -149
    up = torch.full((1, 4), 3e38, device="cuda")
    codes, _ = mlb.CudaSiluMulInt8DeviceInput(gate.float(), up)
    assert codes.tolist() == [[102, 76, 25, 127]]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_small_beside_large(cuda, rows, n, dtype):
    t = getattr(torch, dtype)
    least = -149 if dtype == "float32" else -133  # the smallest number's exponent
    g = torch.Generator(device="cuda").manual_seed(rows * n)

    def rand(lo, hi):
        return torch.rand(rows, n, device="cuda", generator=g, dtype=torch.float64) * (hi - lo) + lo

    sign = torch.where(rand(0, 1) < 0.5, -1.0, 1.0)
    few = torch.floor(rand(1, 100)) * 2.0 ** least * sign  # a few of the smallest steps
    around = 2.0 ** rand(-130, -122) * sign  # either side of the smallest normal number
    large = 2.0 ** rand(100, 127)
    for gate, up in ((few, torch.full_like(few, 3e38)), (few, large), (around, large),
                     (large, few), (large, around)):  # the second's gates' reciprocals are 1
        check(gate.to(t), up.to(t))
    # beside ordinary products, and alone against them
    gate, up = few.clone(), large.clone()
    gate[:, ::3] = rand(-4, 4)[:, ::3]
    up[:, ::3] = 2.0 ** rand(-60, -20)[:, ::3]
    check(gate.to(t), up.to(t))
