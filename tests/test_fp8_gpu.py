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


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 4, 5, 6, 7])
@pytest.mark.parametrize("N", [61, 64, 67, 126, 137, 264, 521])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_results_at_any_address(offset, N, dtype):
    """Rows that begin anywhere in a 16-byte word, as a result's does that lies within a buffer: the same bits as in a buffer of its own, and nothing beside it."""
    from piccl_b200.ops import fp8
    M, K = 203, 256
    a, b = fp8.empty(M, K), fp8.empty(N, K)
    fp8.quantize(_randn(M, K, seed=1), a)
    fp8.quantize(_randn(N, K, seed=2), b)
    wide = fp8.empty((N + 7) // 8 * 8, K)
    fp8.quantize(torch.cat([_randn(N, K, seed=2), torch.zeros(-N % 8, K, dtype=torch.bfloat16, device="cuda")]), wide)
    want = torch.empty(M, (N + 7) // 8 * 8, dtype=dtype, device="cuda")
    fp8.product(a, wide, want)
    for tile in (64, 128, 256):
        buf = torch.full((M * N + 16,), math.nan, dtype=dtype, device="cuda")
        fp8.product(a, b, buf[offset:offset + M * N].view(M, N), _tile=min(tile, 128) if dtype == torch.float32 else tile)
        assert torch.equal(buf[offset:offset + M * N].view(M, N), want[:, :N])
        assert bool(buf[:offset].isnan().all()) and bool(buf[offset + M * N:].isnan().all())


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


# ------------------------------------------------------------------ what a caller may pass
def test_values_that_are_not_finite():
    """They become NaN and leave the scales of their block, row and square to the others."""
    from piccl_b200.ops import fp8
    for dtype in (torch.bfloat16, torch.float32):
        x = _randn(200, 300, seed=1, dtype=dtype)
        x[3, 5], x[130, 200], x[131, 299] = math.nan, math.inf, -math.inf
        x[7, 128:256] = math.inf
        x[8, :128] = 0
        for square in (False, True):
            q, t = fp8.empty(200, 300), fp8.empty(300, 200)
            fp8.quantize(x, q, transposed=t, square=square)
            _same(q, x, square)
            _same(t, x.t(), square)
            r = fp8.empty(200, 300)
            fp8.quantize(x, r, square=square)
            assert torch.equal(r.values.view(torch.uint8), q.values.view(torch.uint8)) and torch.equal(r.scales, q.scales)
    # a product: rows and columns that hold them, and no others
    a, w = fp8.empty(200, 300), fp8.empty(72, 300)
    fp8.quantize(x, a)
    fp8.quantize(_randn(72, 300, seed=2), w)
    y = torch.empty(200, 72, dtype=torch.bfloat16, device="cuda")
    fp8.product(a, w, y)
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    bad[[3, 7, 130, 131]] = True
    assert torch.equal(y.isnan().all(1), bad) and torch.equal(y.isnan().any(1), bad)
    for m in (1, 8, 16):                                          # and where the kernel of few rows rounds
        part = x[128:128 + m].to(torch.bfloat16).contiguous()
        z = torch.empty(m, 72, dtype=torch.bfloat16, device="cuda")
        fp8.linear(part, w, z)
        fp8.quantize(part, (b := fp8.empty(m, 300)))
        want = fp8.dequantize(b) @ fp8.dequantize(w).t()
        assert torch.equal(z.isnan(), want.isnan())


@pytest.mark.parametrize("scale", [2.0 ** -130, 2.0 ** -126, 2.0 ** -110, 2.0 ** 100, 2.0 ** 120])
def test_the_ends_of_the_range(scale):
    from piccl_b200.ops import fp8
    x = _randn(130, 257, seed=3, dtype=torch.float32).clamp(-8, 8) * scale * 16
    for square in (False, True):
        q, t = fp8.empty(130, 257), fp8.empty(257, 130)
        fp8.quantize(x, q, transposed=t, square=square)
        _same(q, x, square)
        _same(t, x.t(), square)


@pytest.mark.parametrize("M,N,K", [(1, 64, 256), (8, 5000, 264), (16, 256, 512), (24, 128, 1024), (200, 256, 1280)])
@pytest.mark.parametrize("up,down", [(120, -30), (-30, 120), (110, -118), (-118, 110), (-60, -50)])
def test_products_of_large_and_small_scales(M, N, K, up, down):
    """The scale of one operand may be far above 1 where the other's is far below: the bound is that of any product."""
    from piccl_b200.ops import fp8
    x, w = _randn(M, K, seed=1, scale=2.0 ** up), _randn(N, K, seed=2, scale=2.0 ** down)
    q, w8 = fp8.empty(M, K), fp8.empty(N, K)
    fp8.quantize(x, q)
    fp8.quantize(w, w8)
    a, b = ((t.values.double() * torch.exp2(fp8.exponents(t).double() - 127).repeat_interleave(128, 1)) for t in (q, w8))
    want, size = a @ b.t(), a.abs() @ b.t().abs()
    for dtype, eps in ((torch.bfloat16, EPS16), (torch.float32, EPS32)):
        y, z = (torch.empty(M, N, dtype=dtype, device="cuda") for _ in range(2))
        fp8.linear(x, w8, y)
        fp8.product(q, w8, z)
        for got in (y, z):
            assert bool(((got.double() - want).abs() <= 2 * EPS32 * (K / 32 + 10) * size + eps * want.abs()).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset,extra", [(0, 0), (1, 0), (0, 3), (8, 8), (3, 16)])
def test_strided_rows_at_any_address(dtype, offset, extra):
    """Rows of a wider matrix that begin in the middle of a 16-byte word, through the quantiser and each kind of layer."""
    from piccl_b200.ops import fp8
    for M, N, K in ((5, 72, 264), (40, 130, 264), (200, 264, 264)):
        wide = _randn(M, K + extra + offset, seed=M, dtype=dtype)
        x = wide[:, offset:offset + K]
        q, p = fp8.empty(M, K), fp8.empty(M, K)
        fp8.quantize(x, q)
        fp8.quantize(x.contiguous(), p)
        assert torch.equal(q.values.view(torch.uint8), p.values.view(torch.uint8)) and torch.equal(q.scales, p.scales)
        w = fp8.empty(N, K)
        fp8.quantize(_randn(N, K, seed=9, scale=0.05), w, square=True)
        y, z = (torch.empty(M, N, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        fp8.linear(x, w, y)
        fp8.product(p, w, z)
        want = fp8.dequantize(p).double() @ fp8.dequantize(w).double().t()
        size = fp8.dequantize(p).double().abs() @ fp8.dequantize(w).double().abs().t()
        for got in (y, z):
            assert bool(((got.double() - want).abs() <= EPS16 * want.abs() + 2 * EPS32 * (K / 32 + 10) * size).all())


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 200, 72), (64, 128, 256), (77, 130, 300), (300, 257, 520), (2331, 768, 264)])
@pytest.mark.parametrize("dw_dtype", [torch.bfloat16, torch.float32])
def test_layer_forward_and_backward(M, N, K, dw_dtype):
    """A layer's three products against the formulas in 64 bits on the rounded operands (whose copies in both directions stand for one matrix), and its gradients against differences of that function:
    it is linear in the input and in the weights, so a difference quotient is exact up to fp64's rounding."""
    from piccl_b200 import ops
    from piccl_b200.ops import fp8
    x, w, dy = _randn(M, K, seed=1), _randn(N, K, seed=2, scale=0.05, dtype=torch.float32), _randn(M, N, seed=3, scale=1e-3)
    w8, w8t, xt = fp8.empty(N, K), fp8.empty(K, N), fp8.empty(K, M)
    fp8.quantize(w, w8, transposed=w8t, square=True)
    assert torch.equal(fp8.dequantize(w8, K), fp8.dequantize(w8t, N).t())
    y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    bias = _randn(N, seed=4)
    assert fp8.linear(x, w8, y, bias=bias, keep=xt) is y
    q, qt, t = fp8.empty(M, K), fp8.empty(K, M), fp8.empty(N, M)
    fp8.quantize(x, q, transposed=qt)
    assert torch.equal(xt.values.view(torch.uint8), qt.values.view(torch.uint8)) and torch.equal(xt.scales, qt.scales)
    dx, dw = torch.empty(M, K, dtype=torch.bfloat16, device="cuda"), torch.empty(N, K, dtype=dw_dtype, device="cuda")
    fp8.linear_bwd(dy, xt, w8t, dx, dw)
    g = fp8.empty(M, N)
    fp8.quantize(dy, g, transposed=t)
    ops.raise_if_a_wait_ran_out()
    wd, xr, xc = fp8.dequantize(w8, K).double(), fp8.dequantize(q, K).double(), fp8.dequantize(xt, M).double().t()
    gr, gc = fp8.dequantize(g, N).double(), fp8.dequantize(t, M).double().t()

    def near(got, want, size, terms):
        half = EPS16 if got.dtype == torch.bfloat16 else EPS32
        assert bool(((got.double() - want).abs() <= half * want.abs() + 2 * EPS32 * (terms / 32 + 10) * size).all())

    near(y, xr @ wd.t() + bias.double(), xr.abs() @ wd.abs().t() + bias.double().abs(), K)
    near(dx, gr @ wd, gr.abs() @ wd.abs(), N)
    near(dw, gc.t() @ xc, gc.abs().t() @ xc.abs(), M)
    # differences of L = sum(g * (x w^T)) along one direction of each argument
    gen = torch.Generator(device="cuda").manual_seed(7)
    for grad, base, f in ((gr @ wd, xr, lambda z: (gr * (z @ wd.t())).sum()), (gc.t() @ xc, wd, lambda z: (gc * (xc @ z.t())).sum())):
        d = torch.randn(base.shape, generator=gen, device="cuda", dtype=torch.float64)
        quotient, size = (f(base + d) - f(base - d)) / 2, (grad.abs() * d.abs()).sum()
        assert abs(quotient - (grad * d).sum()) <= 1e-9 * size + 1e-30
    # one of the two alone
    dx2, dw2 = torch.empty_like(dx), torch.empty_like(dw)
    fp8.linear_bwd(dy, None, w8t, dx2, None)
    fp8.linear_bwd(dy, xt, None, None, dw2)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


def test_empty_operands_and_sums_over_nothing():
    from piccl_b200.ops import fp8
    bias = _randn(72)
    w = fp8.empty(72, 128)
    fp8.quantize(_randn(72, 128), w)
    y = torch.full((0, 72), math.nan, dtype=torch.bfloat16, device="cuda")
    assert fp8.linear(_randn(0, 128), w, y, bias=bias, keep=fp8.empty(128, 0)) is y
    none, x0 = fp8.empty(72, 0), torch.empty(5, 0, dtype=torch.bfloat16, device="cuda")
    y = torch.full((5, 72), math.nan, dtype=torch.bfloat16, device="cuda")
    fp8.linear(x0, none, y, bias=bias)
    assert torch.equal(y, bias.expand(5, 72))
    fp8.linear(x0, none, y)
    assert not y.any()
    dx, dw = torch.full((0, 128), math.nan, dtype=torch.bfloat16, device="cuda"), torch.full((72, 128), math.nan, device="cuda")
    fp8.linear_bwd(torch.empty(0, 72, dtype=torch.bfloat16, device="cuda"), fp8.empty(128, 0), fp8.empty(128, 72), dx, dw)
    assert not dw.any()


def test_refusals_on_the_gpu():
    from piccl_b200.ops import fp8
    x, w, y = _randn(4, 128), fp8.empty(8, 128), torch.empty(4, 8, dtype=torch.bfloat16, device="cuda")
    fp8.quantize(_randn(8, 128), w)
    for call in (lambda: fp8.quantize(x, None), lambda: fp8.quantize(x, fp8.empty(5, 128)), lambda: fp8.quantize(x, fp8.empty(4, 256)), lambda: fp8.quantize(x, fp8.empty(4, 128), fp8.empty(4, 128)),
                 lambda: fp8.quantize(x, fp8.empty(4, 128, "cpu")), lambda: fp8.quantize(x.t(), fp8.empty(128, 4)), lambda: fp8.quantize(x.double(), fp8.empty(4, 128)),
                 lambda: fp8.linear(x, fp8.empty(8, 256), y), lambda: fp8.linear(x, w, y[:3]), lambda: fp8.linear(x, w, y.t()), lambda: fp8.linear(x, w, y.half()), lambda: fp8.linear(x, w, y.cpu()),
                 lambda: fp8.linear(x, w, y, bias=torch.zeros(8, device="cuda")), lambda: fp8.linear(x, w, y, bias=_randn(9)), lambda: fp8.linear(x, w, y, keep=fp8.empty(4, 128)),
                 lambda: fp8.product(w, w, y), lambda: fp8.product(fp8.Fp8(w.values, w.scales[:0]), w, torch.empty(8, 8, device="cuda")), lambda: fp8.product(fp8.Fp8(w.values.view(torch.uint8), w.scales), w, y),
                 lambda: fp8.linear_bwd(y, None, None, None, torch.empty(8, 128, device="cuda")), lambda: fp8.linear_bwd(y, fp8.empty(128, 300), None, None, torch.empty(8, 128, device="cuda")),
                 lambda: fp8.linear_bwd(y, None, w, torch.empty(4, 128, dtype=torch.bfloat16, device="cuda"), None)):
        with pytest.raises(ValueError):
            call()


def test_results_that_overlap_operands_are_refused():
    """In place a block of a launch would write what another has yet to read."""
    from piccl_b200.ops import fp8
    x, w, wt = _randn(4, 128), fp8.empty(128, 128), fp8.empty(128, 128)
    fp8.quantize(_randn(128, 128), w, transposed=wt, square=True)
    q, xt, y, dw = fp8.empty(4, 128), fp8.empty(128, 4), torch.zeros_like(x), torch.empty(128, 128, dtype=torch.bfloat16, device="cuda")
    fp8.quantize(x, q, transposed=xt)
    row = torch.zeros(1, 128, dtype=torch.bfloat16, device="cuda")
    q1 = fp8.empty(1, 128)
    fp8.quantize(row, q1)
    inside = xt.values.view(torch.bfloat16)[:8].view(4, 128)          # room within xt
    assert inside.data_ptr() == xt.values.data_ptr()
    before = x.clone()
    for call in (lambda: fp8.linear(x, w, x), lambda: fp8.linear(row, w, row), lambda: fp8.product(q1, w, row, bias=row[0]), lambda: fp8.product(q, w, w.values.view(torch.bfloat16)[:8].view(4, 128)),
                 lambda: fp8.quantize(x, q, transposed=fp8.Fp8(xt.values, q.scales)), lambda: fp8.quantize(x, fp8.Fp8(x.view(fp8.E4M3)[:2].view(4, 128), q.scales)),
                 lambda: fp8.linear_bwd(y, xt, wt, y, dw), lambda: fp8.linear_bwd(y, xt, wt, inside, dw), lambda: fp8.linear_bwd(y, xt, wt, dw[:4], dw)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert torch.equal(x, before)


def test_calls_close_on_each_other_streams_and_graphs():
    """Results of calls that nothing waits between, of two streams at a time and of a captured layer and its backward pass are those of calls one by one."""
    from piccl_b200 import ops
    from piccl_b200.ops import fp8
    shapes = [(1, 520, 1024), (12, 264, 512), (24, 264, 2048), (50, 136, 640), (300, 520, 384)]
    sets = []
    for i, (M, N, K) in enumerate(shapes):
        x, dy = _randn(M, K, seed=i), _randn(M, N, seed=10 + i)
        w8, w8t = fp8.empty(N, K), fp8.empty(K, N)
        fp8.quantize(_randn(N, K, seed=20 + i, scale=0.05), w8, transposed=w8t, square=True)
        sets.append((x, dy, w8, w8t, M, N, K))

    def step(s):
        x, dy, w8, w8t, M, N, K = s
        out = [torch.empty(M, N, dtype=torch.bfloat16, device="cuda"), torch.empty(M, N, dtype=torch.bfloat16, device="cuda"), torch.empty(M, K, dtype=torch.bfloat16, device="cuda"),
               torch.empty(N, K, device="cuda")]
        xt = fp8.empty(K, M)
        fp8.linear(x, w8, out[0])
        fp8.linear(x, w8, out[1], keep=xt)
        fp8.linear_bwd(dy, xt, w8t, out[2], out[3])
        return out

    want = []
    for s in sets:
        want.append(step(s))
        torch.cuda.synchronize()
    for _ in range(20):
        got = [step(s) for s in sets]
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                results.append([step(s) for s in sets])
    torch.cuda.synchronize()
    for got in results:
        for a, b in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = [step(s) for s in sets]
        graphs.append((g, out))
    for _ in range(3):
        for g, out in graphs:
            for o in out:
                for t in o:
                    t.fill_(math.nan)
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            for a, b in zip(want, out):
                assert all(torch.equal(p, q) for p, q in zip(a, b))
    ops.raise_if_a_wait_ran_out()


def test_the_calls_through_ctypes_give_the_same():
    """Where Python's headers are missing, calls go through ctypes."""
    from piccl_b200.ops import fp8
    from piccl_b200.ops.optimizer import AdamW
    results = []
    kept = fp8._native_calls()
    for native in (True, False):
        fp8._fast = kept if native else False
        try:
            out = []
            for M, N, K in ((4, 72, 264), (70, 136, 300)):
                x, dy = _randn(M, K, seed=1), _randn(M, N, seed=2)
                w8, w8t, xt = fp8.empty(N, K), fp8.empty(K, N), fp8.empty(K, M)
                fp8.quantize(_randn(N, K, seed=3), w8, transposed=w8t, square=True)
                y, z, dx, dw = (torch.empty(*s, dtype=torch.bfloat16, device="cuda") for s in ((M, N), (M, N), (M, K), (N, K)))
                fp8.linear(x, w8, y, bias=_randn(N, seed=4))
                fp8.linear(x, w8, z, keep=xt)
                fp8.linear_bwd(dy, xt, w8t, dx, dw)
                out += [y, z, dx, dw]
            p, g = torch.ones(300, device="cuda"), _randn(300, seed=5, dtype=torch.float32)
            opt = AdamW([p], [g], bits=8)
            opt.step(1e-2, gscale=0.5)
            opt.step(1e-2, gscale=torch.full((1,), 0.5, device="cuda"))
            results.append([*out, p, opt.m.float(), opt.v.float(), opt.step_dev])
        finally:
            fp8._fast = kept
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_training_a_layer_in_8_bits():
    """The operators together, as a program would use them: round the weights, forward, backward, the optimiser with moments in 8 bits, for some steps; against the same steps put together from plain
    operations in fp64 on what the kernels rounded."""
    from piccl_b200.ops import fp8
    from piccl_b200.ops.optimizer import AdamW
    M, N, K = 96, 264, 392
    w = _randn(N, K, seed=1, scale=0.05, dtype=torch.float32)
    p = w.to(torch.bfloat16)
    dw = torch.empty(N, K, dtype=torch.bfloat16, device="cuda")
    opt = AdamW([p], [dw], [w], bits=8, seed=3)
    w8, w8t, xt = fp8.empty(N, K), fp8.empty(K, N), fp8.empty(K, M)
    y, dx = torch.empty(M, N, dtype=torch.bfloat16, device="cuda"), torch.empty(M, K, dtype=torch.bfloat16, device="cuda")
    for step in range(1, 4):
        x, target = _randn(M, K, seed=10 + step), _randn(M, N, seed=20 + step)
        fp8.quantize(p, w8, transposed=w8t, square=True)
        fp8.linear(x, w8, y, keep=xt)
        dy = (y - target) / M
        fp8.linear_bwd(dy, xt, w8t, dx, dw)
        before, (m, v) = w.double(), [t.double() for t in opt.moments(0)]
        opt.step(1e-3, 0.9, 0.95, 1e-8, 0.1)
        g = dw.double().view(-1)
        size = 1e-3 * (0.9 * m.abs() + 0.1 * g.abs()) / (1 - 0.9 ** step)          # the sum that gives m may cancel, its addends' roundings do not
        m, v = 0.9 * m + 0.1 * g, 0.95 * v + 0.05 * g * g
        below = (v / (1 - 0.95 ** step)).sqrt() + 1e-8
        want = before.view(-1) * (1 - 1e-4) - 1e-3 * (m / (1 - 0.9 ** step)) / below
        # some 16 half steps of that (counted at _reference of the optimiser's tests), two of the weight
        assert bool(((w.double().view(-1) - want).abs() <= 2 * EPS32 * (before.view(-1).abs() + want.abs() + 10 * size / below)).all())
        assert torch.equal(p, w.to(torch.bfloat16))
        fp8.quantize(dy, (q := fp8.empty(M, N)))
        d, size = fp8.dequantize(q, N).double() @ fp8.dequantize(w8, K).double(), fp8.dequantize(q, N).double().abs() @ fp8.dequantize(w8, K).double().abs()
        assert bool(((dx.double() - d).abs() <= EPS16 * d.abs() + 2 * EPS32 * (N / 32 + 10) * size).all())
