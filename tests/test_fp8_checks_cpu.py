"""What the 8-bit layers and the optimiser refuse (no GPU needed: nothing is launched)."""
import ctypes as C

import pytest
import torch

BF = torch.bfloat16


def _fp8(rows, cols):
    from piccl_b200.ops import fp8
    return fp8.empty(rows, cols, "cpu")


def test_room_and_order_of_scales():
    from piccl_b200.ops import fp8
    a = _fp8(130, 513)
    assert tuple(a.values.shape) == (130, 640) and tuple(a.scales.shape) == (2, 2, 32, 4, 4)
    a.scales.copy_(torch.arange(a.scales.numel()).view(a.scales.shape) % 251)
    e = fp8.exponents(a)
    for r, k in ((0, 0), (31, 3), (32, 1), (127, 4), (129, 2)):
        assert e[r, k] == a.scales[r // 128, k // 4, r % 32, r // 32 % 4, k % 4]
    a.values.copy_(torch.ones(130, 640).to(fp8.E4M3))
    assert torch.equal(fp8.dequantize(a, 513)[:, 512], torch.exp2(e[:, 4].float() - 127))


@pytest.mark.parametrize("x,out,transposed,why", [
    (torch.zeros(4, 4, dtype=torch.float16), (4, 4), None, "matrix"), (torch.zeros(4, dtype=BF), (4, 4), None, "matrix"), (torch.zeros(4, 8, dtype=BF)[:, ::2], (4, 4), None, "next to each other"),
    (torch.zeros(4, 4, dtype=BF), (4, 4), None, "CUDA"), (torch.zeros(4, 4, dtype=BF).expand(4, 4).t(), (4, 4), None, "next to each other"),
    (torch.zeros(1, 4, dtype=BF).expand(3, 4), (3, 4), None, "next to each other")])
def test_quantize_refuses(x, out, transposed, why):
    from piccl_b200.ops import fp8
    with pytest.raises(ValueError, match=why):
        fp8.quantize(x, _fp8(*out), transposed)


def test_products_refuse():
    from piccl_b200.ops import fp8
    a, b, out = _fp8(4, 128), _fp8(8, 128), torch.zeros(4, 8, dtype=BF)
    for bad in (out[:, ::2], out.to(torch.float16), out[0], out):
        with pytest.raises(ValueError):
            fp8.product(a, b, bad)
    with pytest.raises(ValueError):
        fp8.linear(torch.zeros(4, 128, dtype=BF), _fp8(8, 256), out)
    with pytest.raises(ValueError):
        fp8.linear_bwd(torch.zeros(4, 8, dtype=BF), None, None, None, torch.zeros(8, 128))


def test_what_overlaps():
    from piccl_b200.ops.fp8 import _check_apart
    x = torch.zeros(8, 16)
    _check_apart("f", [x[:4], None], [x[4:], x[:0]])
    _check_apart("f", [x[0]], [x[1:, :3], x[0, :0]])
    for written, read in (([x[:4]], [x[3:]]), ([x[:4], x[3:5]], []), ([x[2]], [x[:, :1]]), ([x], [None, x.view(torch.int16)[5:6]])):
        with pytest.raises(ValueError, match="overlap"):
            _check_apart("f", written, read)


def test_native_entries_refuse_before_they_touch_an_address():
    from piccl_b200 import _native as N
    from piccl_b200.ops import fp8
    lib, p, good = N.ops_lib(), C.c_void_p, 4096
    quant, gemm = lib.piccl_ops_fp8_quantize, lib.piccl_ops_fp8_gemm
    quant.argtypes, gemm.argtypes = fp8._QUANTIZE, fp8._GEMM
    ok = [good, 0, 16, 16, 16, good, good, good, good, 0, 0]
    for at, bad, rc in ((0, 0, -2), (0, good + 1, -2), (2, 0, -1), (3, 0, -1), (4, 15, -1), (5, 0, -2), (6, 0, -2), (5, good + 8, -2), (7, 0, -2), (8, good + 4, -2)):
        assert quant(*[bad if i == at else x for i, x in enumerate(ok)]) == rc, (at, bad)
    assert quant(good, 0, 16, 16, 16, 0, 0, 0, 0, 0, 0) == -2
    ok = [good, good, good, good, 0, good, 0, 16, 16, 128, 0, 0]
    for at, bad, rc in ((0, 0, -2), (1, good + 8, -2), (2, good + 4, -2), (3, 0, -2), (4, good + 1, -2), (5, 0, -2), (5, good + 1, -2), (7, 0, -1), (8, -1, -1), (9, 64, -1), (9, 0, -1)):
        assert gemm(*[bad if i == at else x for i, x in enumerate(ok)]) == rc, (at, bad)


def test_adamw_refuses():
    from piccl_b200.ops.optimizer import _STEP, AdamW
    f, b = torch.zeros(8), torch.zeros(8, dtype=BF)
    for args, kw, why in (([[b], [b]], {}, "master"), ([[f], [b], [f]], {}, "master"), ([[f], [b]], {"bits": 16}, "bits"), ([[], []], {}, "parameters"), ([[f], [b, b]], {}, "gradients"),
                          ([[b], [b], [torch.zeros(7)]], {}, "master"), ([[f], [b]], {}, "CUDA"), ([[f], [b]], {"decay": [True, False]}, "decays")):
        with pytest.raises(ValueError, match=why):
            AdamW(*args, **kw)
    from piccl_b200 import _native as N
    step = N.ops_lib().piccl_ops_adamw_many
    step.argtypes = _STEP
    good = 4096
    ok = [good, good, 1, 1, good, good, good, good, 1e-3, 0.9, 0.95, 1e-8, 0.1, 1.0, 0, good, good, 0, 0]
    for at, bad, rc in ((0, 0, -2), (1, 0, -2), (2, -1, -1), (4, 0, -2), (4, good + 8, -2), (4, good + 16, -2), (5, good + 4, -2), (6, 0, -2), (7, 0, -2), (9, 1.0, -1), (9, -0.1, -1), (10, 1.5, -1), (15, 0, -2), (16, 0, -2)):
        assert step(*[bad if i == at else x for i, x in enumerate(ok)]) == rc, (at, bad)
