"""Products of 8-bit operands over long sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS16, EPS32 = 2.0 ** -8, 2.0 ** -24          # half a step of bf16 and of fp32, relative to the value


@pytest.mark.parametrize("M,N,K", [(200, 264, 32768), (1, 264, 32768), (24, 128, 32768), (300, 130, 131072)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("signs", ["random", "one"])
def test_long_sums(M, N, K, dtype, signs):
    """The tensor cores cut their fp32 sums off where an fma would round them: each step of 32 k loses up to a unit in the last place of what has been added so far, 2^-23 of it, which is at most 2^-23 of the sum of
    magnitudes.  Sums of one sign lose the most: the partial sums grow evenly, so K / 32 steps lose K / 64 units at most."""
    from piccl_b200 import ops
    from piccl_b200.ops import fp8
    gen = torch.Generator(device="cuda").manual_seed(K + M)
    a, b = fp8.empty(M, K), fp8.empty(N, K)
    for to, rows in ((a, M), (b, N)):
        x = torch.randn(rows, K, generator=gen, device="cuda")
        fp8.quantize(x.abs() if signs == "one" else x, to)
    x, y = fp8.dequantize(a).double(), fp8.dequantize(b).double()
    want, size = x @ y.t(), x.abs() @ y.t().abs()
    out = torch.empty(M, N, dtype=dtype, device="cuda")
    fp8.product(a, b, out)
    ops.raise_if_a_wait_ran_out()
    off, half = (out.double() - want).abs(), EPS16 if dtype == torch.bfloat16 else EPS32
    print("beyond the result's own rounding, of the sum of magnitudes, in steps of 2^-24:", float(((off - half * want.abs()) / (EPS32 * size)).max()))
    steps = K / 32 if signs == "random" else K / 64
    assert bool((off <= half * want.abs() + 2 * EPS32 * (steps + 10) * size).all())
