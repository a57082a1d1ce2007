"""Linear layers in 8 bits: the quantiser and the products of src/ops/fp8_quant.cu, fp8_gemm.cu and, for few rows, fp8_few.cu.

A matrix in 8 bits (`Fp8`) is e4m3 values, rows filled with zeros to a multiple of 128, and one power of two for each block of 128
values of a row: byte e, 1 to 254, stands for 2^(e - 127), the smallest for which the block's largest finite magnitude is at most 448.  Values that
are not finite become NaN.  A product sums along the rows of both operands, so a matrix that two products sum over different
dimensions is kept twice, the second time transposed; `square` gives both copies of a weight the same values.

    w8, w8t = fp8.empty(N, K), fp8.empty(K, N)
    fp8.quantize(w, w8, transposed=w8t, square=True)         # after each optimiser step
    xt = fp8.empty(K, M)
    fp8.linear(x, w8, y, bias=b, keep=xt)                    # y = x w^T + b; xt is what the backward pass needs of x, at a byte an element
    fp8.linear_bwd(dy, xt, w8t, dx, dw)                      # dx = dy w, dw = dy^T x

Sums are fp32 in the tensor cores, which cut off where an fma would round: each step of 32 k loses up to 2^-23 of the sum so far, always toward zero.  Results in fp32 are added up, rounded, from sums of 1024 k;
those in bf16 are one sum over all of k, which is too small by up to 2^-23 K / 64 of it where all addends have one sign (1.5e-5 at K = 8192, beside the 2e-3 of a rounding to bf16), and with random signs by some
2^-25 K / 48 of a result's usual size.  Results are rounded once.  Calls launch on the current stream of their tensors' device, take workspace from PyTorch's
allocator, and can be captured.  Results overlap neither operands nor each other.  Empty results are left alone; a sum over nothing is zero (or the bias).
"""
from __future__ import annotations

import ctypes as C
from contextlib import nullcontext
from typing import NamedTuple, Optional, Sequence

import torch

from .. import _native as N
from . import _bump, _s
from .gemm_sm100 import _native, _ptr

E4M3 = torch.float8_e4m3fn
_QUANTIZE = [C.c_void_p, C.c_int] + [C.c_longlong] * 3 + [C.c_void_p] * 4 + [C.c_int, C.c_void_p]
_GEMM = [C.c_void_p] * 6 + [C.c_int] * 3 + [C.c_longlong, C.c_int, C.c_void_p]
_SCRATCH = [C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_longlong, C.c_int]
_LINEAR = [C.c_void_p, C.c_int, C.c_longlong] + [C.c_void_p] * 4 + [C.c_int] + [C.c_void_p] * 4 + [C.c_int] * 2 + [C.c_longlong, C.c_void_p]
_fast = None


def _native_calls():
    """The calls as one native function each (src/python/tensorcall.cc), or False where Python's headers are missing: a layer through ctypes is 23 us of host time, through it 5."""
    global _fast
    if _fast is None:
        _fast = N.tensorcall() or False
    return _fast


class Fp8(NamedTuple):
    """values: e4m3 [rows, columns up to a multiple of 128]; scales: uint8 [ceil(rows / 128), ceil(blocks / 4), 32, 4, 4], block k of row r at
    [r // 128, k // 4, r % 32, r // 32 % 4, k % 4], the order in which the tensor cores take them."""
    values: torch.Tensor
    scales: torch.Tensor


def empty(rows: int, cols: int, device="cuda") -> Fp8:
    """Room for a matrix of `rows` by `cols`."""
    fast = _native_calls()
    if fast and (t := fast.empty(rows, cols, device)):
        return Fp8(*t)
    blocks = (cols + 127) // 128
    return Fp8(torch.empty(rows, blocks * 128, dtype=E4M3, device=device), torch.empty((rows + 127) // 128, (blocks + 3) // 4, 32, 4, 4, dtype=torch.uint8, device=device))


def exponents(a: Fp8) -> torch.Tensor:
    """The bytes of the scales as [rows, blocks]."""
    s = a.scales
    return s.permute(0, 3, 2, 1, 4).reshape(s.shape[0] * 128, s.shape[1] * 4)[:a.values.shape[0], :a.values.shape[1] // 128]


def dequantize(a: Fp8, cols: Optional[int] = None) -> torch.Tensor:
    """What the matrix stands for, in fp32 (its first `cols` columns)."""
    v = torch.ldexp(a.values.float(), (exponents(a).to(torch.int32) - 127).repeat_interleave(128, 1))
    return v if cols is None else v[:, :cols]


def _on(device: torch.device):
    return nullcontext() if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _check_fp8(a: Fp8, name: str, device) -> None:
    v, s = a
    if v.dim() != 2 or v.dtype != E4M3 or not v.is_contiguous() or v.shape[1] % 128:
        raise ValueError(f"{name}: contiguous e4m3 values of whole blocks of 128 wanted, got {v.dtype} {tuple(v.shape)}")
    if s.dtype != torch.uint8 or not s.is_contiguous() or tuple(s.shape) != ((v.shape[0] + 127) // 128, (v.shape[1] + 511) // 512, 32, 4, 4):
        raise ValueError(f"{name}: the scales are not those of {tuple(v.shape)} values: {s.dtype} {tuple(s.shape)}")
    if v.device != device or s.device != device:
        raise ValueError(f"{name}: tensors of one CUDA device wanted")


def _check_matrix(x: torch.Tensor, name: str, dtypes, contiguous: bool) -> None:
    if x.dim() != 2 or x.dtype not in dtypes:
        raise ValueError(f"{name}: a matrix of {' or '.join(str(t)[6:] for t in dtypes)} wanted, got {x.dtype} {tuple(x.shape)}")
    if (contiguous and not x.is_contiguous()) or (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        raise ValueError(f"{name}: rows of values next to each other wanted, got strides {x.stride()}")
    if not x.is_cuda:
        raise ValueError(f"{name}: tensors of one CUDA device wanted")


def _check_apart(name: str, written: Sequence[Optional[torch.Tensor]], read: Sequence[Optional[torch.Tensor]]) -> None:
    """What is written shares no bytes with what is read, nor with what else is written: blocks of a launch read operands while others write."""
    bytes_of = lambda t: (t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size())  # noqa: E731
    w, r = ([bytes_of(t) for t in ts if t is not None and t.numel()] for ts in (written, read))
    if any(a[0] < b[1] and b[0] < a[1] for i, a in enumerate(w) for b in w[i + 1:] + r):
        raise ValueError(f"{name}: operands and results that overlap")


def _done(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed (code {rc})")
    _bump()


def quantize(x: torch.Tensor, out: Optional[Fp8], transposed: Optional[Fp8] = None, square: bool = False) -> None:
    """x [R, C], bf16 or fp32, -> out, blocks along its rows (room for R x C), and transposed, blocks along its columns (room for C x R), either of which may be None.
    square: one power of two for each 128 x 128 values."""
    fast = _native_calls()
    if fast and (n := fast.quantize(x, out, transposed, square)):
        _bump(n)
        return
    _check_matrix(x, "quantize", (torch.bfloat16, torch.float32), False)
    if out is None and transposed is None:
        raise ValueError("quantize: nothing to write")
    R, Cc = x.shape
    for a, rows, cols in ((out, R, Cc), (transposed, Cc, R)):
        if a is not None:
            _check_fp8(a, "quantize", x.device)
            if tuple(a.values.shape) != (rows, (cols + 127) // 128 * 128):
                raise ValueError(f"quantize: room for {rows} x {cols} wanted, got {tuple(a.values.shape)}")
    _check_apart("quantize", [*(out or ()), *(transposed or ())], [x])
    if R == 0 or Cc == 0:
        for a in (out, transposed):
            if a is not None:
                a.scales.fill_(1)
        return
    with _on(x.device):
        q, t = out or (None, None), transposed or (None, None)
        _done(_native("piccl_ops_fp8_quantize", _QUANTIZE)(x.data_ptr(), x.dtype == torch.float32, R, Cc, x.stride(0) if R > 1 else Cc, _ptr(q[0]), _ptr(q[1]), _ptr(t[0]), _ptr(t[1]), square, _s()),
              "fp8 quantize")


def _check_product(a: tuple, b: Fp8, out: torch.Tensor, bias) -> None:
    _check_matrix(out, "product", (torch.bfloat16, torch.float32), True)
    _check_fp8(b, "product", out.device)
    (M, K), Nn = a, b.values.shape[0]
    if b.values.shape[1] != K or tuple(out.shape) != (M, Nn):
        raise ValueError(f"product: [{M}, {K}] and [{Nn}, {b.values.shape[1]}] do not give {tuple(out.shape)}")
    if bias is not None and (bias.dtype != torch.bfloat16 or tuple(bias.shape) != (Nn,) or not bias.is_contiguous() or bias.device != out.device):
        raise ValueError(f"product: a bias of {Nn} bf16 wanted, got {bias.dtype} {tuple(bias.shape)}")


def product(a: Fp8, b: Fp8, out: torch.Tensor, bias: Optional[torch.Tensor] = None, _tile: int = 0) -> torch.Tensor:
    """out [M, N] (bf16 or fp32) = a [M, K] b [N, K]^T + bias [N] (bf16)"""
    fast = _native_calls()
    if fast and not _tile and (n := fast.product(a, b, out, bias)):
        _bump(n)
        return out
    _check_fp8(a, "product", out.device)
    _check_product(tuple(a.values.shape), b, out, bias)
    _check_apart("product", [out], [*a, *b, bias])
    (M, K), Nn = a.values.shape, b.values.shape[0]
    if M == 0 or Nn == 0:
        return out
    if K == 0:
        return out.zero_() if bias is None else out.copy_(bias.expand(M, Nn))
    with _on(out.device):
        _done(_native("piccl_ops_fp8_gemm", _GEMM)(a.values.data_ptr(), a.scales.data_ptr(), b.values.data_ptr(), b.scales.data_ptr(), _ptr(bias), out.data_ptr(), out.dtype == torch.float32, M, Nn, K,
                                                   _tile, _s()), "fp8 product")
    return out


def linear(x: torch.Tensor, w: Fp8, out: torch.Tensor, bias: Optional[torch.Tensor] = None, keep: Optional[Fp8] = None) -> torch.Tensor:
    """out [M, N] = x [M, K] w [N, K]^T + bias, x (bf16 or fp32) rounded to 8 bits on the way; keep: room for K x M, receives x along the tokens for linear_bwd."""
    fast = _native_calls()
    if fast and (n := fast.linear(x, w, out, bias, keep)):
        _bump(n)
        return out
    _check_matrix(x, "linear", (torch.bfloat16, torch.float32), False)
    M, K = x.shape
    _check_apart("linear", [out, *(keep or ())], [x, *w, bias])
    if w.values.dim() != 2 or w.values.shape[1] != (K + 127) // 128 * 128:
        raise ValueError(f"linear: weights of {K} columns wanted, got {tuple(w.values.shape)}")
    _check_product((M, w.values.shape[1]), w, out, bias)          # all of it before anything is written
    if out.device != x.device:
        raise ValueError("linear: tensors of one CUDA device wanted")
    if keep is None and K and 0 < M <= 32 and not _native("piccl_ops_fp8_linear_scratch", _SCRATCH)(x.data_ptr(), x.dtype == torch.float32, x.stride(0) if M > 1 else K, M, w.values.shape[0], K, False):
        if out.numel() == 0:
            return out
        with _on(x.device):
            rc = _native("piccl_ops_fp8_linear", _LINEAR)(x.data_ptr(), False, x.stride(0) if M > 1 else K, w.values.data_ptr(), w.scales.data_ptr(), _ptr(bias), out.data_ptr(),
                                                          out.dtype == torch.float32, None, None, None, None, M, out.shape[1], K, _s())
            _done(min(rc, 0), "fp8 linear")
        return out
    q = empty(M, K, x.device)
    quantize(x, q, keep)
    return product(q, w, out, bias)


def linear_bwd(dy: torch.Tensor, xt: Optional[Fp8], wt: Optional[Fp8], dx: Optional[torch.Tensor], dw: Optional[torch.Tensor]) -> None:
    """dx [M, K] = dy [M, N] w, from the weights' transposed copy wt (K x N); dw [N, K] = dy^T x, from the input along the tokens xt (K x M).  dy (bf16 or fp32) is rounded to 8 bits, along
    both dimensions in one pass.  dx or dw may be None."""
    fast = _native_calls()
    if fast and (n := fast.linear_bwd(dy, xt, wt, dx, dw)):
        _bump(n)
        return
    _check_matrix(dy, "linear_bwd", (torch.bfloat16, torch.float32), False)
    if dx is None and dw is None:
        return
    if (dx is not None and wt is None) or (dw is not None and xt is None):
        raise ValueError("linear_bwd: dx takes the transposed weights, dw the input along the tokens")
    M, Nn = dy.shape
    _check_apart("linear_bwd", [dx, dw], [dy, *(xt or ()), *(wt or ())])
    for a, n in ((wt if dx is not None else None, Nn), (xt if dw is not None else None, M)):
        if a is not None and (a.values.dim() != 2 or a.values.shape[1] != (n + 127) // 128 * 128):
            raise ValueError(f"linear_bwd: {n} columns wanted, got {tuple(a.values.shape)}")
    for b, out, rows in ((wt, dx, M), (xt, dw, Nn)):
        if out is not None:                                           # all of it before anything is written
            _check_product((rows, b.values.shape[1]), b, out, None)
            if out.device != dy.device:
                raise ValueError("linear_bwd: tensors of one CUDA device wanted")
    q = empty(M, Nn, dy.device) if dx is not None else None
    t = empty(Nn, M, dy.device) if dw is not None else None
    quantize(dy, q, t)
    if dx is not None:
        product(q, wt, dx)
    if dw is not None:
        product(t, xt, dw)
