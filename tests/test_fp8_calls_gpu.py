"""The 8-bit layers' calls, natively and through ctypes: one behaviour, and what a refused or failed call leaves behind."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "ctypes"])
def path(request, monkeypatch):
    """Each call path in turn (ctypes: as where Python's headers are missing)"""
    from piccl_b200.ops import fp8
    if request.param == "ctypes":
        monkeypatch.setattr(fp8, "_fast", False)
    else:
        assert fp8._native_calls()
    return request.param


def _randn(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def test_out_of_memory_is_pytorchs_own_error(path):
    """Programs catch that type to free caches or to shrink a batch."""
    from piccl_b200.ops import fp8
    with pytest.raises(torch.OutOfMemoryError):
        fp8.empty(1 << 24, 1 << 20, torch.device("cuda", 0))          # 16 TiB
    M, N, K = 8192, 256, 4096
    x, w, wt, xt = _randn(M, K), fp8.empty(N, K), fp8.empty(K, N), fp8.empty(K, M)
    fp8.quantize(_randn(N, K, seed=1), w, transposed=wt, square=True)
    fp8.quantize(x, None, transposed=xt)
    y, dx, dw = (torch.empty(*s, dtype=torch.bfloat16, device="cuda") for s in ((M, N), (M, K), (N, K)))
    dy = _randn(M, N, seed=2)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved() / total, 0)
    held = []
    try:
        for size in (1 << 25, 1 << 22, 1 << 21, 1 << 19):          # what is reserved but free
            with pytest.raises(torch.OutOfMemoryError):
                while True:
                    held.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
        with pytest.raises(torch.OutOfMemoryError):
            fp8.linear(x, w, y)
        with pytest.raises(torch.OutOfMemoryError):
            fp8.linear_bwd(dy, xt, wt, dx, dw)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, 0)
    held.clear()
    fp8.linear(x, w, y)
    q = fp8.empty(M, K)
    fp8.quantize(x, q)
    want = fp8.product(q, w, torch.empty_like(y))
    assert torch.equal(y, want)


def test_refused_calls_write_nothing(path):
    """A call with one argument that is not as it has to be leaves the others alone, whichever it is."""
    from piccl_b200.ops import fp8
    M, N, K = 40, 72, 264
    x, dy, w, wt, xt = _randn(M, K), _randn(M, N), fp8.empty(N, K), fp8.empty(K, N), fp8.empty(K, M)
    fp8.quantize(_randn(N, K, seed=1), w, transposed=wt, square=True)
    fp8.quantize(x, None, transposed=xt)
    y, dx, dw = (torch.full(s, 7.0, dtype=torch.bfloat16, device="cuda") for s in ((M, N), (M, K), (N, K)))
    keep = fp8.empty(K, M)
    keep.values.view(torch.uint8).fill_(5)
    keep.scales.fill_(9)
    bias = _randn(N)
    for call in (lambda: fp8.linear(x, w, y, bias=bias[:9], keep=keep), lambda: fp8.linear(x, w, y.half(), keep=keep), lambda: fp8.linear(x, w, y[:9], keep=keep), lambda: fp8.linear(x, w, y.cpu(), keep=keep),
                 lambda: fp8.linear(x, fp8.Fp8(w.values, w.scales[:0]), y, keep=keep), lambda: fp8.linear(x, w, y, bias=bias.cpu(), keep=keep), lambda: fp8.linear(x, w, y, keep=fp8.Fp8(keep.values, keep.scales[:1])),
                 lambda: fp8.linear_bwd(dy, xt, wt, dx, dw.half()), lambda: fp8.linear_bwd(dy, xt, wt, dx, dw[:9]), lambda: fp8.linear_bwd(dy, xt, wt, dx, dw.cpu()), lambda: fp8.linear_bwd(dy, xt, wt, dx.t(), dw),
                 lambda: fp8.linear_bwd(dy, fp8.Fp8(xt.values, xt.scales[:1]), wt, dx, dw), lambda: fp8.linear_bwd(dy, xt, fp8.Fp8(wt.values.view(torch.uint8), wt.scales), dx, dw)):
        with pytest.raises(ValueError):
            call()
        assert all(bool((t == 7.0).all()) for t in (y, dx, dw)) and bool((keep.values.view(torch.uint8) == 5).all()) and bool((keep.scales == 9).all())
