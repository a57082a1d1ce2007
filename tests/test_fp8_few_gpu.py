"""Layers of few rows in one launch, which rounds the input itself (src/ops/fp8_few.cu), against the quantiser and a product in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS16, EPS32 = 2.0 ** -8, 2.0 ** -24          # half a step of bf16 and of fp32, relative to the value


def _randn(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _one_launch(x, n):
    from piccl_b200.ops import fp8
    from piccl_b200.ops.gemm_sm100 import _native
    return not _native("piccl_ops_fp8_linear_scratch", fp8._SCRATCH)(x.data_ptr(), x.dtype == torch.float32, x.stride(0) if x.shape[0] > 1 else x.shape[1], x.shape[0], n, x.shape[1], False)


def _check(x, N, dtype, w_at=None):
    """The layer of x with weights of N rows (one value of which is not finite, if w_at says where) and a bias: NaN where the row of x or of the weights holds what is not finite, the others within the bound of sums in
    fp32 of eight warps (at each step of 32 a rounding, doubled for additions that cut off) and the result's own rounding."""
    from piccl_b200.ops import fp8
    M, K = x.shape
    assert _one_launch(x, N)
    wf = _randn(N, K, seed=3, scale=0.02)
    if w_at is not None:
        wf[w_at] = -math.inf
    w, q, bias = fp8.empty(N, K), fp8.empty(M, K), _randn(N, seed=4)
    fp8.quantize(wf, w)
    fp8.quantize(x, q)
    guard = torch.full((M + 1, N), 7.0, dtype=dtype, device="cuda")
    fp8.linear(x, w, guard[:M], bias=bias)
    a, b = fp8.dequantize(q).double(), fp8.dequantize(w).double()
    assert torch.equal(a.isnan().any(1), ~x.isfinite().all(1)) and torch.equal(b.isnan().any(1), ~wf.isfinite().all(1))
    want, size = a @ b.t() + bias.double(), a.abs() @ b.abs().t() + bias.double().abs()
    bad = (~x.isfinite().all(1))[:, None] | (~wf.isfinite().all(1))[None, :]
    got = guard[:M].double()
    assert torch.equal(got.isnan(), bad) and torch.equal(want.isnan(), bad)
    bound = 2 * EPS32 * (K / 32 + 2 + 8) * size + (EPS16 if dtype == torch.bfloat16 else EPS32) * want.abs()
    assert bool(((got - want).abs() <= bound)[~bad].all())
    assert bool((guard[M] == 7.0).all())


@pytest.mark.parametrize("M", [1, 2, 5, 8, 9, 16])
@pytest.mark.parametrize("N,K", [(72, 304), (1000, 128), (257, 1016)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_not_finite_stays_in_its_row(M, N, K, dtype):
    for value in (math.inf, -math.inf, math.nan):
        for row, col in {(0, 0), (M // 2, K // 2), (M - 1, K - 1)}:
            x = _randn(M, K, seed=1) * torch.exp(_randn(M, 1, seed=2) * 2)
            x[row, col] = value
            _check(x, N, dtype)
    x = _randn(M, K, seed=1)
    x[M - 1, :128] = math.inf                       # a block that is nothing else
    x[0, K - 8:] = math.nan
    _check(x, N, dtype, w_at=(N // 2, K // 3))
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[M // 2, 5] = -math.inf                        # beside zeros alone
    _check(x, N, dtype)


@pytest.mark.parametrize("M", [1, 2, 4])
@pytest.mark.parametrize("N,K", [(5000, 2312), (5000, 4096), (4737, 2056), (9473, 2824)])
def test_wide_weights_of_more_blocks_than_are_under_way(M, N, K):
    """32 rows of the weights to a block, whose warps have two blocks of 128 each under way and load the later ones as they go."""
    x = _randn(M, K, seed=M) * torch.exp(_randn(M, 1, seed=2) * 2)
    _check(x, N, torch.bfloat16)
    x[M - 1, K - 200] = math.nan
    _check(x, N, torch.float32, w_at=(N - 1, K - 1))


@pytest.mark.parametrize("M,N,K", [(1, 520, 4360), (3, 136, 4360), (2, 40, 8192)])
def test_narrow_weights_of_more_blocks_than_are_under_way(M, N, K):
    """16 rows of the weights to a block, four blocks of 128 to a warp under way."""
    x = _randn(M, K, seed=M)
    _check(x, N, torch.bfloat16)
    x[0, 4224] = math.inf
    _check(x, N, torch.float32)
