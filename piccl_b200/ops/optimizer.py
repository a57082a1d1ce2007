"""AdamW over many tensors in one launch (src/ops/adamw_many.cu), moments in fp32 or in 8 bits.

    opt = AdamW(params, grads, masters, bits=8, decay=[p.dim() > 1 for p in params])
    opt.step(lr, b1, b2, eps, wd)

Parameters are bf16 with an fp32 master each, or fp32 with none; gradients are bf16 or fp32; tensors are contiguous, of any size and at any address.
`decay` says which of them decay (all, by default).  The number of steps done lives on the device (`step_dev`, advanced by each step), so that a
step can be captured into a CUDA graph and replayed; `gscale` multiplies the gradients, and may be a device tensor (a clipping factor that nobody reads back).

Moments are the optimiser's own: `m` and `v`, flat, each tensor from a multiple of 128 elements on (`places`).  In 8 bits they are e4m3 values with
a power of two for each block of 128 (`m_scales`, `v_scales`: byte e stands for 2^(e - 127)), v as its root, and are rounded stochastically, by bits that
depend on the element's place, the step and `seed` alone: 2.02 bytes a parameter in place of 8 (and 0.03 for the table that tells each block's tensor).  Values that are not finite are held as NaN.

What 8 bits cost: each held value is within a step of e4m3 (6 to 12 %) of the one that it stands for, and right in the mean.  The square of a root that is right in the mean is too large by the rounding's
variance: at most 13.5 % in the mean of v, 2.5 % measured at b2 = 0.95 and 3.4 % at 0.999 (gradients of one size); an element's root has a deviation of 12 to 16 %, 98 % of them are between 0.73 and 1.4 times the exact one.  The random bits
of a place at one step are those of the place after it at the step before: an element's own roundings are independent from step to step, but the errors of neighbours' roots go together (correlation 0.3 to 0.46 from
one element to the next, over some 1 / (1 - b2) elements; none in m, where signs differ).
These tensors, `step_dev` and `seed` are what captured steps go on reading and cannot be exchanged: a state is loaded into them (`load_state`, or `opt.m.copy_(...)`).  Parameters, masters and gradients stay where
they are too; a step after one of them has been given other memory (`p.data = ...`) is refused.

One step at a time: steps of one optimiser on several streams need the order that any two writers of the same tensors need.
"""
from __future__ import annotations

import ctypes as C
from bisect import bisect
from typing import Mapping, Optional, Sequence, Union

import torch

from . import _bump, _s
from .fp8 import E4M3, _native_calls, _on
from .gemm_sm100 import _native, _ptr

_DECAY, _P_F32, _G_F32, _WORDS = 1, 2, 4, 8
_STEP = [C.c_void_p, C.c_void_p, C.c_longlong, C.c_int] + [C.c_void_p] * 4 + [C.c_float, C.c_double, C.c_double] + [C.c_float] * 3 + [C.c_void_p] * 3 + [C.c_uint, C.c_void_p]


class _Tensor(C.Structure):          # AdamTensor of src/ops/adamw_many.cu
    _fields_ = [("p", C.c_void_p), ("master", C.c_void_p), ("g", C.c_void_p), ("n", C.c_longlong), ("block", C.c_longlong), ("flags", C.c_int), ("pad", C.c_int)]


class AdamW:
    def __init__(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], masters: Optional[Sequence[torch.Tensor]] = None, bits: int = 32,
                 decay: Optional[Sequence[bool]] = None, seed: int = 0):
        if bits not in (8, 32):
            raise ValueError(f"AdamW: moments of 8 or 32 bits, not {bits}")
        params, grads = list(params), list(grads)
        masters = [None] * len(params) if masters is None else list(masters)
        decay = [True] * len(params) if decay is None else list(decay)
        if not params or not len(params) == len(grads) == len(masters) == len(decay):
            raise ValueError(f"AdamW: {len(params)} parameters, {len(grads)} gradients, {len(masters)} masters, {len(decay)} decays")
        self._device = params[0].device
        for p, w in zip(params, masters):
            if p.dtype not in (torch.bfloat16, torch.float32) or (p.dtype == torch.float32) != (w is None):
                raise ValueError("AdamW: parameters are bf16 with a master or fp32 without")
            if w is not None and (w.dtype != torch.float32 or w.numel() != p.numel()):
                raise ValueError(f"AdamW: an fp32 master of {p.numel()} elements wanted, got {w.dtype} {tuple(w.shape)}")
            for t in (p,) if w is None else (p, w):
                if not t.is_contiguous() or not t.is_cuda or t.device != self.device:
                    raise ValueError("AdamW: contiguous tensors of one CUDA device wanted")
        written = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (*params, *(w for w in masters if w is not None)) if t.numel())
        if any(a[1] > b[0] for a, b in zip(written, written[1:])):
            raise ValueError("AdamW: parameters or masters that overlap")
        self._written = written
        self._params, self._masters, self._decay, self._bits, self._seed = tuple(params), tuple(masters), tuple(bool(d) for d in decay), bits, int(seed) & 0xFFFFFFFF
        self._fixed = [(t, t.data_ptr()) for t in (*params, *masters) if t is not None]
        places, block = [], 0                         # (first element in m and v, elements) of each tensor
        for p in params:
            places.append((block * 128, p.numel()))
            block += (p.numel() + 127) // 128
        self._places, self._blocks = tuple(places), block
        zeros = lambda n, dtype: torch.zeros(n, dtype=dtype, device=self.device)  # noqa: E731
        kind = E4M3 if bits == 8 else torch.float32
        self._m, self._v = zeros(block * 128, kind), zeros(block * 128, kind)
        self._m_scales, self._v_scales = (torch.ones(block, dtype=torch.uint8, device=self.device) for _ in range(2)) if bits == 8 else (None, None)
        self._step_dev, self._ticket = zeros(1, torch.int32), zeros(1, torch.int32)
        lengths = [(n + 127) // 128 for _, n in self.places if n]
        self._owner = torch.repeat_interleave(torch.arange(len(lengths), dtype=torch.int32), torch.tensor(lengths, dtype=torch.int64)).to(self.device)      # the tensor of each block
        self._table = None
        self._calls = _native_calls()
        self._fast = self._calls.adamw_step if self._calls else None
        self.set_grads(grads)

    # what the table and the native handle were made from, and captured steps go on reading: not to be set
    (device, params, masters, grads, decay, bits, seed, places, blocks, m, v, m_scales, v_scales, step_dev) = (
        property(lambda self, name=name: getattr(self, name)) for name in ("_device", "_params", "_masters", "_grads", "_decay", "_bits", "_seed", "_places", "_blocks", "_m", "_v", "_m_scales", "_v_scales", "_step_dev"))

    def state(self) -> dict[str, torch.Tensor]:
        """The optimiser's own tensors, by name: what has to be kept, beside the parameters and masters, to go on with the next step."""
        names = ("m", "v", "step_dev", *(("m_scales", "v_scales") if self.bits == 8 else ()))
        return {name: getattr(self, name) for name in names}

    def load_state(self, state: Mapping[str, torch.Tensor]) -> None:
        """Takes over the values of another's `state`: of as many bits, over tensors of the same sizes (and made with the same `seed`, if its steps are to be repeated bit by bit)."""
        mine = self.state()
        for name, t in mine.items():
            if name not in state or state[name].dtype != t.dtype or state[name].shape != t.shape:
                raise ValueError(f"AdamW: {name} of {t.numel()} {t.dtype} wanted, got {'none' if name not in state else (state[name].dtype, tuple(state[name].shape))}")
        for name, t in mine.items():
            t.copy_(state[name])

    @staticmethod
    def _stay(tensors) -> None:
        if any(t.data_ptr() != at for t, at in tensors):
            raise ValueError("AdamW: a parameter, master or gradient is not where it was (it has been given other memory)")

    def set_grads(self, grads: Sequence[torch.Tensor]) -> None:
        """Other tensors to take the gradients from, from the next step on (a copy of addresses to the device; not within a capture)."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"AdamW: {len(self.params)} gradients wanted, got {len(grads)}")
        with _on(self.device):                        # the stream that the copy goes to
            capturing = torch.cuda.is_current_stream_capturing()
        if capturing:
            raise RuntimeError("AdamW: gradients cannot be exchanged within a capture")
        self._stay(self._fixed)
        records = []
        for p, w, g, d, (first, n) in zip(self.params, self.masters, grads, self.decay, self.places):
            if g.dtype not in (torch.bfloat16, torch.float32) or g.numel() != n or not g.is_contiguous() or g.device != self.device:
                raise ValueError(f"AdamW: a contiguous gradient of {n} elements, bf16 or fp32, on {self.device} wanted, got {g.dtype} {tuple(g.shape)} on {g.device}")
            if n == 0:
                continue
            at = bisect(self._written, (g.data_ptr() + n * g.element_size() - 1, 1 << 64)) - 1      # the last of them that begins before the gradient's end
            if at >= 0 and self._written[at][1] > g.data_ptr():
                raise ValueError("AdamW: a gradient that overlaps a parameter or a master")
            flags = _DECAY * d | _P_F32 * (w is None) | _G_F32 * (g.dtype == torch.float32)
            if all(t is None or t.data_ptr() % (8 * t.element_size()) == 0 for t in (p, w, g)):
                flags |= _WORDS
            records.append(_Tensor(p.data_ptr(), 0 if w is None else w.data_ptr(), g.data_ptr(), n, first // 128, flags, 0))
        self._grads = tuple(grads)
        raw = torch.frombuffer(bytearray((_Tensor * max(1, len(records)))(*records)), dtype=torch.uint8)
        if self._table is None:
            self._table = raw.to(self.device)
        else:
            self._table.copy_(raw)                    # in place: captured steps read it, and steps before on this stream have
        self._stand = self._fixed + [(g, g.data_ptr()) for g in grads]
        if self._calls:
            self._handle = self._calls.adamw(self.device.index, self._table.data_ptr(), self._owner.data_ptr(), self.blocks, self.bits == 8, self.m.data_ptr(), self.v.data_ptr(), _ptr(self.m_scales) or 0,
                                             _ptr(self.v_scales) or 0, self.step_dev.data_ptr(), self._ticket.data_ptr(), self.seed, tuple(t for t, _ in self._stand))

    def step(self, lr: float, b1: float = 0.9, b2: float = 0.95, eps: float = 1e-8, wd: float = 0.1, gscale: Union[float, torch.Tensor] = 1.0) -> None:
        """One step from the gradients as they are now."""
        if self._fast is not None and self._fast(self._handle, lr, b1, b2, eps, wd, gscale):
            _bump()
            return
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: decay rates of the moments are in [0, 1), not {b1} and {b2}")
        dev = None
        if isinstance(gscale, torch.Tensor):
            if gscale.dtype != torch.float32 or gscale.numel() != 1 or gscale.device != self.device:
                raise ValueError("AdamW: gscale is a number or one fp32 value on the device of the parameters")
            gscale, dev = 1.0, gscale
        self._stay(self._stand)
        with _on(self.device):
            rc = _native("piccl_ops_adamw_many", _STEP)(self._table.data_ptr(), self._owner.data_ptr(), self.blocks, self.bits == 8, self.m.data_ptr(), self.v.data_ptr(), _ptr(self.m_scales),
                                                        _ptr(self.v_scales), lr, b1, b2, eps, wd, gscale, _ptr(dev), self.step_dev.data_ptr(), self._ticket.data_ptr(), self.seed, _s())
        if rc != 0:
            raise RuntimeError(f"adamw_many failed (code {rc})")
        _bump()

    def moments(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        """m and v of tensor i as they are held, in fp32."""
        o, n = self.places[i]
        if self.bits == 32:
            return self.m[o:o + n].clone(), self.v[o:o + n].clone()
        out = []
        for values, scales in ((self.m, self.m_scales), (self.v, self.v_scales)):
            k = (n + 127) // 128
            x = torch.ldexp(values[o:o + k * 128].float().view(k, 128), scales[o // 128:o // 128 + k, None].to(torch.int32) - 127)
            out.append(x.reshape(-1)[:n])
        return out[0], out[1] * out[1]
