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
