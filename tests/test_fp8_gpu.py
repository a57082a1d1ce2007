"""The 8-bit format, its quantiser and its products against plain implementations in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS16, EPS32 = 2.0 ** -8, 2.0 ** -24          # half a step of bf16 and of fp32, relative to the value


def _randn(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _quantized(x, square):
    """(values as they stand in e4m3, exponents) of the rows of x in blocks of 128, or of squares, from the definition in fp64"""
    x = x.double()
    r, c = x.shape
    full = torch.nn.functional.pad(x, (0, -c % 128, 0, -r % 128))
    t = full.view(full.shape[0] // 128, 128, full.shape[1] // 128, 128)
    fin = torch.where(t.isfinite(), t.abs(), 0.0)
    top = fin.amax((1, 3), keepdim=True).expand(-1, 128, -1, -1) if square else fin.amax(3, keepdim=True)
    s = torch.ceil(torch.log2(top / 448)).clamp(min=-126.0)
    s = torch.where(top > 448 * torch.exp2(s), s + 1, torch.where(top <= 448 * torch.exp2(s - 1), s - 1, s)).clamp(min=-126.0)      # log2 may be off by its last bit
    y = t * torch.exp2(-s)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    q = torch.where(t.isfinite(), torch.round(y / step) * step, math.nan)
    e = (s + 127).reshape(full.shape[0], -1)
    e[r:] = 1
    return q.reshape(full.shape)[:r], e


def _same(a, x, square):
    from piccl_b200.ops import fp8
    q, e = _quantized(x, square)
    got = a.values.double()
    assert torch.equal(got.isnan(), q.isnan())
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(q))
    k = e.shape[1]
    all_bytes = a.scales.permute(0, 3, 2, 1, 4).reshape(a.scales.shape[0] * 128, -1).double()
    assert torch.equal(all_bytes[:, :k], e) and bool((all_bytes[:, k:] == 1).all())
    assert torch.equal(fp8.exponents(a).double(), e[:x.shape[0]])


SHAPES = [(1, 1), (1, 128), (3, 129), (127, 65), (128, 128), (129, 512), (200, 1000), (513, 640), (1000, 72)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("copies", ["rows", "transposed", "both"])
def test_quantize(rows, cols, dtype, square, copies):
    from piccl_b200.ops import fp8
    x = _randn(rows, cols, seed=rows + cols, dtype=dtype) * torch.exp(_randn(rows, 1, seed=5, dtype=torch.float32) * 3).to(dtype)
    q = fp8.empty(rows, cols) if copies != "transposed" else None
    t = fp8.empty(cols, rows) if copies != "rows" else None
    fp8.quantize(x, q, transposed=t, square=square)
    if q is not None:
        _same(q, x, square)
    if t is not None:
        _same(t, x.t(), square)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 256, 128), (128, 128, 128), (256, 256, 512), (255, 257, 384), (300, 520, 1000), (129, 64, 4096), (2331, 768, 200), (64, 50257, 768), (1000, 72, 640), (48, 1000, 2048), (33, 97, 1152)])
@pytest.mark.parametrize("tile", [0, 64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_product(M, N, K, tile, dtype):
    """Products of e4m3 values have at most 8 bits, so every addend is exact; the sum is fp32.  Allowed: a rounding by 2^-24 of the sum of magnitudes for each step of 32, doubled for
    additions that cut off in place of rounding, and the result's own rounding."""
    from piccl_b200 import ops
    from piccl_b200.ops import fp8
    a, b = fp8.empty(M, K), fp8.empty(N, K)
    fp8.quantize(_randn(M, K, seed=1) * torch.exp(_randn(M, 1, seed=2) * 2), a)
    fp8.quantize(_randn(N, K, seed=3, scale=0.02), b)
    bias = _randn(N, seed=4) if M % 2 else None
    guard = torch.full((M + 1, N), math.nan, device="cuda", dtype=dtype)
    fp8.product(a, b, guard[:M], bias=bias, _tile=min(tile, 128) if dtype == torch.float32 else tile)
    x, y = fp8.dequantize(a).double(), fp8.dequantize(b).double()
    want, size = x @ y.t(), x.abs() @ y.t().abs()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    off = (guard[:M].double() - want).abs()
    bound = 2 * EPS32 * (K / 32 + 2) * size + (EPS16 if dtype == torch.bfloat16 else EPS32) * want.abs()
    print("worst share of the bound", float((off / bound.clamp(min=1e-300)).max()), "sum in steps of 2^-24", float((off / (EPS32 * size).clamp(min=1e-300)).max()))
    ops.raise_if_a_wait_ran_out()
    assert bool((off <= bound).all())
    assert torch.isnan(guard[M]).all()


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 15, 16, 17, 23, 25, 31, 32, 33, 64, 65])
@pytest.mark.parametrize("N,K", [(1, 8), (128, 128), (257, 640), (1000, 1096), (4096, 1024), (520, 4104), (136, 72), (64, 333), (5000, 264), (64, 8192)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_of_few_rows(M, N, K, dtype):
    """One launch up to 64 rows where they lie on 16-byte boundaries: the same bits as the quantiser and a product in 64 bits, within that product's bound."""
    from piccl_b200 import ops
    from piccl_b200.ops import fp8
    x = _randn(M, K, seed=M) * torch.exp(_randn(M, 1, seed=2) * 2)
    w, q = fp8.empty(N, K), fp8.empty(M, K)
    fp8.quantize(_randn(N, K, seed=3, scale=0.02), w, square=True)
    fp8.quantize(x, q)
    bias = _randn(N, seed=4) if M % 2 else None
    a, b = fp8.dequantize(q).double(), fp8.dequantize(w).double()
    want, size = a @ b.t(), a.abs() @ b.t().abs()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    bound = 2 * EPS32 * (K / 32 + 2 + 8) * size + (EPS16 if dtype == torch.bfloat16 else EPS32) * want.abs()          # sums of up to 8 slices
    for call in ("linear", "product"):
        guard = torch.full((M + 1, N), math.nan, device="cuda", dtype=dtype)
        if call == "linear":
            fp8.linear(x, w, guard[:M], bias=bias)
        else:
            fp8.product(q, w, guard[:M], bias=bias)
        ops.raise_if_a_wait_ran_out()
        assert bool(((guard[:M].double() - want).abs() <= bound).all()), call
        assert torch.isnan(guard[M]).all()
