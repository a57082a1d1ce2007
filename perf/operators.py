"""Training in 8 bits: linear layers whose products run on e4m3 operands with a power of two for each block of 128 values, the
quantiser that writes those operands, and AdamW over many tensors with its moments in 32 or in 8 bits.

The format, common to all: a block of 128 values along a row (or a square of 128 x 128) has one byte e, its values are
q * 2^(e - 127) with q in e4m3, e the smallest for which the block's largest finite magnitude stays within 448.  Rows are padded
with zeros to whole blocks.  Scales lie as [rows / 128, blocks / 4, 32, 4, 4], row r and block k at [r // 128, k // 4, r % 32, r // 32 % 4, k % 4].
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # activations of a training step of 8 x 1024 tokens, as they are kept for the backward pass: along the rows and along the tokens
        {"name": "quantize_activations", "op": "quantize", "rows": 8192, "cols": 4096, "dtype": "bf16", "square": False, "both": True},
        # the embedding table of GPT-2 medium after an optimiser step, from its fp32 masters: squares, and the transposed copy that the input gradient takes
        {"name": "quantize_embedding", "op": "quantize", "rows": 50257, "cols": 1024, "dtype": "fp32", "square": True, "both": True},
        # a single token through a layer of GPT-2 medium: latency and the weights' bytes
        {"name": "linear_one_token", "op": "linear", "m": 1, "n": 4096, "k": 1024, "bias": True, "keep": False},
        # a few sequences' next tokens through the layer back
        {"name": "linear_few_tokens", "op": "linear", "m": 24, "n": 1024, "k": 4096, "bias": True, "keep": False},
        # the head of a mid-size model on a ragged batch: an odd number of columns, rows no multiple of any tile
        {"name": "linear_head_ragged", "op": "linear", "m": 2331, "n": 50257, "k": 768, "bias": False, "keep": False},
        # a layer of GPT-2 medium in training: the input is kept in 8 bits for the weights' gradient
        {"name": "linear_training", "op": "linear", "m": 8192, "n": 4096, "k": 1024, "bias": True, "keep": True},
        # the product of the benchmark of the tensor-parallel kernels: compute bound
        {"name": "linear_large", "op": "linear", "m": 8192, "n": 8192, "k": 3584, "bias": False, "keep": False},
        # backward pass on a ragged batch, the weights' gradient in fp32 as an accumulating program wants it
        {"name": "backward_ragged", "op": "backward", "m": 2331, "n": 2304, "k": 768, "dw": "fp32"},
        # backward pass of GPT-2 medium's second MLP layer
        {"name": "backward_training", "op": "backward", "m": 8192, "n": 1024, "k": 4096, "dw": "bf16"},
        # the smallest model's parameters: launch latency
        {"name": "adamw_tiny", "op": "adamw", "bits": 8, "layers": 2, "d_model": 256, "vocab": 1000, "seq": 128, "ragged": 0, "master": False, "grad": "fp32", "step": 0},
        # all parameters of GPT-2 medium, moments in 32 bits
        {"name": "adamw_medium_32", "op": "adamw", "bits": 32, "layers": 24, "d_model": 1024, "vocab": 50257, "seq": 1024, "ragged": 0, "master": True, "grad": "bf16", "step": 99},
        # the same with moments in 8 bits
        {"name": "adamw_medium_8", "op": "adamw", "bits": 8, "layers": 24, "d_model": 1024, "vocab": 50257, "seq": 1024, "ragged": 0, "master": True, "grad": "bf16", "step": 99},
    ]


# ------------------------------------------------------------------ drawing
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "linear", "backward", "backward", "adamw", "adamw", "adamw"])
    if op == "quantize":
        c = {"op": op, "rows": _log(rng, 1, 50304), "cols": rng.choice([256, 768, 1024, 4096, _log(rng, 1, 8192)]), "dtype": rng.choice(["bf16", "bf16", "fp32"]),
             "square": rng.random() < 0.4, "both": rng.random() < 0.6}
        while c["rows"] * c["cols"] > 50257 * 1024:
            c["rows"] = (c["rows"] + 1) // 2
        return c
    if op == "adamw":
        c = {"op": op, "bits": rng.choice([8, 8, 32]), "layers": rng.randint(2, 24), "d_model": rng.choice([256, 512, 768, 1024]), "vocab": _log(rng, 1000, 50257), "seq": rng.choice([128, 777, 1024]),
             "ragged": 0, "master": rng.random() < 0.6, "grad": rng.choice(["bf16", "fp32"]), "step": rng.choice([0, 1, 10, 1000, 20000])}
        if rng.random() < 0.4:          # many tensors of any size, one element among them
            c |= {"layers": 0, "d_model": 0, "vocab": 0, "seq": 0, "ragged": rng.randint(1, 1 << 20)}
        return c
    if op == "linear":
        m = rng.choice([1, 2, rng.randint(3, 16), rng.randint(17, 128), _log(rng, 129, 8192), _log(rng, 129, 8192), 4096])
    else:
        m = rng.choice([_log(rng, 1, 8192), _log(rng, 128, 8192), 4096])
    n = rng.choice([1024, 2048, 4096, 2304, _log(rng, 16, 8192), _log(rng, 16, 8192)])
    k = rng.choice([1024, 2048, 4096, 768, _log(rng, 16, 8192), _log(rng, 16, 8192)])
    while 2 * m * n * k > 2 * 8192 * 8192 * 3584:
        m = (m + 1) // 2
    if op == "linear":
        return {"op": op, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5, "keep": m > 16 and rng.random() < 0.4}
    return {"op": op, "m": m, "n": n, "k": k, "dw": rng.choice(["bf16", "fp32"])}


# ------------------------------------------------------------------ the format, in elementary operations
def _up(n, d):
    return (n + d - 1) // d


def _byte(amax):
    return (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=1)


def _finite(x):
    return torch.where(torch.isfinite(x), x.abs(), 0.0)


def _power(byte):
    """2^(127 - byte)"""
    return ((254 - byte) << 23).view(torch.float32)


def _order(byte):
    """[rows, blocks] -> the order in which scales lie; what is beyond the matrix is a block of zeros, whose byte is 1"""
    r, k = byte.shape
    full = torch.ones(_up(r, 128) * 128, _up(k, 4) * 4, dtype=torch.uint8, device=byte.device)
    full[:r, :k] = byte
    return full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _unorder(scales, rows, blocks):
    t, k4 = scales.shape[:2]
    return scales.permute(0, 3, 2, 1, 4).reshape(t * 128, k4 * 4)[:rows, :blocks].to(torch.int32)


def _padded(x):
    """fp32, rows filled with zeros to whole blocks of 128"""
    p = torch.zeros(x.shape[0], _up(x.shape[1], 128) * 128, dtype=torch.float32, device=x.device)
    p[:, :x.shape[1]] = x
    return p


def _quantize(x, square=False):
    """values [rows, whole blocks] and scales"""
    p = _padded(x)
    r, c = p.shape
    if square:
        t = torch.zeros(_up(r, 128) * 128, c, dtype=torch.float32, device=x.device)
        t[:r] = _finite(p)
        byte = _byte(t.view(-1, 128, c // 128, 128).amax((1, 3))).repeat_interleave(128, 0)[:r]
    else:
        byte = _byte(_finite(p).view(r, -1, 128).amax(2))
    q = p.view(r, -1, 128) * _power(byte)[:, :, None]
    q = torch.where(torch.isfinite(q), q, math.nan)
    return q.view(r, c).to(E4M3), _order(byte)


def _values(q):
    values, scales = q
    r, c = values.shape
    return (values.float().view(r, -1, 128) / _power(_unorder(scales, r, c // 128))[:, :, None]).view(r, c)


# ------------------------------------------------------------------ preparation
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(gen, rows, cols, dtype=torch.bfloat16, std=1.0):
    # a few columns are far larger than the others, as in the residual stream of a trained model
    x = torch.randn(rows, cols, generator=gen, device="cuda") * std
    wide = torch.rand(cols, generator=gen, device="cuda") < 0.01
    return (x * torch.where(wide, 20.0, 1.0)).to(dtype)


def _gradients(gen, rows, cols):
    # rows of very different size
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    return (x * torch.exp(torch.randn(rows, 1, generator=gen, device="cuda") * 2.0 - 10.0)).to(torch.bfloat16)


def _sizes(c):
    """The tensors of a model, those that decay first: the flat order of this file; each begins at a multiple of 128"""
    if c["ragged"]:
        r = random.Random(c["ragged"])
        return [_log(r, 1, 1 << 20) for _ in range(r.randint(1, 40))], [_log(r, 1, 4096) for _ in range(r.randint(1, 80))]
    d, n = c["d_model"], c["layers"]
    decay = [c["vocab"] * d, c["seq"] * d] + [3 * d * d, d * d, 4 * d * d, 4 * d * d] * n
    return decay, [d, d] + [d, d, 3 * d, d, d, d, 4 * d, d] * n


def _flat(sizes):
    off, places = 0, []
    for n in sizes:
        places.append((off, n))
        off += _up(n, 128) * 128
    return off, places


def prepare(case, seed):
    gen = _gen(seed)
    if case["op"] == "quantize":
        x = _activations(gen, case["rows"], case["cols"], TYPES[case["dtype"]], 0.02 if case["square"] else 1.0)
        return {"case": case, "x": x}
    if case["op"] == "linear":
        w = _quantize(torch.randn(case["n"], case["k"], generator=gen, device="cuda") * 0.02, square=True)
        bias = (torch.randn(case["n"], generator=gen, device="cuda") * 0.1).to(torch.bfloat16) if case["bias"] else None
        return {"case": case, "x": _activations(gen, case["m"], case["k"]), "w": w, "bias": bias}
    if case["op"] == "backward":
        w = torch.randn(case["n"], case["k"], generator=gen, device="cuda") * 0.02
        # what the forward pass has left: the input along the tokens, and the transposed copy of the weights
        xt = _quantize(_activations(gen, case["m"], case["k"]).t())
        return {"case": case, "dy": _gradients(gen, case["m"], case["n"]), "wt": _quantize(w.t(), square=True), "xt": xt}
    decay, rest = _sizes(case)
    total, places = _flat(decay + rest)
    border = places[len(decay)][0]
    held = torch.zeros(total, dtype=torch.bool, device="cuda")       # what lies between two tensors stays zero
    ends = torch.tensor([o + n for o, n in places], device="cuda")
    starts = torch.tensor([o for o, _ in places], device="cuda")
    at = torch.arange(total, device="cuda")
    held = at < ends[torch.searchsorted(starts, at, right=True) - 1]
    del at
    size = torch.exp(torch.randn(total // 128, 1, generator=gen, device="cuda") - 9.0).expand(-1, 128).reshape(-1)

    def normal():
        return torch.where(held, torch.randn(total, generator=gen, device="cuda"), 0.0)

    w = normal() * 0.02
    g = (normal() * size).to(TYPES[case["grad"]])
    s = {"case": case, "border": border, "p": w.to(torch.bfloat16) if case["master"] else w, "master": w if case["master"] else None, "g": g,
         "step": torch.full((1,), case["step"], dtype=torch.int32, device="cuda"), "seed": seed & 0x7FFFFFFF, "rates": (3e-4, 0.9, 0.95, 1e-8, 0.1, 0.7)}
    begun = 1.0 if case["step"] else 0.0
    m, r = normal() * size * (0.2 * begun), normal().abs() * size * begun
    if case["bits"] == 32:
        s |= {"m": m, "v": r * r}
    else:
        for name, x in (("m", m), ("v", r)):          # held of the second moment is its root
            x = x.view(-1, 128)
            byte = _byte(x.abs().amax(1))
            s[name] = (x * _power(byte)[:, None]).view(-1).to(E4M3)
            s[name + "_scales"] = byte.to(torch.uint8)
    if own:
        from piccl_b200.ops.optimizer import AdamW
        view = lambda t: None if t is None else [t[o:o + n] for o, n in places]  # noqa: E731
        opt = AdamW(view(s["p"]), view(s["g"]), view(s["master"]), bits=case["bits"], decay=[True] * len(decay) + [False] * len(rest), seed=s["seed"])
        for name in ("m", "v", "m_scales", "v_scales"):
            if name in s:
                getattr(opt, name).copy_(s.pop(name))
        opt.step_dev.copy_(s.pop("step"))
        s["opt"] = opt
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return {"quantize": _run_quantize, "linear": _run_linear, "backward": _run_backward, "adamw": _run_adamw}[state["case"]["op"]](state)


def _run_quantize(s):
    c, x = s["case"], s["x"]
    if own:
        from piccl_b200.ops import fp8
        q = fp8.empty(*x.shape, x.device)
        t = fp8.empty(x.shape[1], x.shape[0], x.device) if c["both"] else None
        fp8.quantize(x, q, transposed=t, square=c["square"])
    else:
        q = _quantize(x, c["square"])
        t = _quantize(x.t(), c["square"]) if c["both"] else None
    return {"rows": list(q), "transposed": list(t) if t else None}


def _run_linear(s):
    c, x = s["case"], s["x"]
    if own:
        from piccl_b200.ops import fp8
        y = torch.empty(c["m"], c["n"], dtype=torch.bfloat16, device=x.device)
        keep = fp8.empty(c["k"], c["m"], x.device) if c["keep"] else None
        fp8.linear(x, fp8.Fp8(*s["w"]), y, bias=s["bias"], keep=keep)
    else:
        y = _values(_quantize(x)) @ _values(s["w"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        y = y.to(torch.bfloat16)
        keep = _quantize(x.t()) if c["keep"] else None
    return {"y": y, "keep": list(keep) if keep else None}


def _run_backward(s):
    c, dy = s["case"], s["dy"]
    if own:
        from piccl_b200.ops import fp8
        dx = torch.empty(c["m"], c["k"], dtype=torch.bfloat16, device=dy.device)
        dw = torch.empty(c["n"], c["k"], dtype=TYPES[c["dw"]], device=dy.device)
        fp8.linear_bwd(dy, fp8.Fp8(*s["xt"]), fp8.Fp8(*s["wt"]), dx, dw)
    else:
        dx = (_values(_quantize(dy)) @ _values(s["wt"]).t()).to(torch.bfloat16)
        dw = (_values(_quantize(dy.t())) @ _values(s["xt"]).t()).to(TYPES[c["dw"]])
    return {"dx": dx, "dw": dw}


def _random(n, seed, step, device):
    """32 random bits for each element: a hash of its place, the seed and the number of the step"""
    key = (seed + step.long() * 0x9E3779B9) & 0xFFFFFFFF
    h = (torch.arange(n, device=device) * 0x9E3779B9 + key) & 0xFFFFFFFF
    h = ((h ^ (h >> 16)) * 0xBB67AE85) & 0xFFFFFFFF
    h = ((h ^ (h >> 15)) * 0x6A09E667) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _stochastic(x, bits16, positive):
    """Blocks of 128 -> e4m3 values (rounded up with the probability of the part cut off) and their bytes; positive: what is not zero stays so"""
    b = x.view(-1, 128)
    byte = _byte(_finite(b).amax(1))
    t = b * _power(byte)[:, None]
    a = t.abs()
    low = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)        # below, steps are those of [2^-6, 2^-5)
    z = (a + low).view(torch.int32) + (bits16.view(-1, 128) << 4).to(torch.int32)
    z = (z & ~0xFFFFF).view(torch.float32) - low
    if positive:
        z = torch.where(a > 0, z.clamp(min=2.0 ** -9), z)
    z = torch.where(torch.isfinite(t), z.copysign(t), math.nan)
    return z.view(-1).to(E4M3), byte.to(torch.uint8)


def _run_adamw(s):
    c = s["case"]
    lr, b1, b2, eps, wd, gscale = s["rates"]
    if own:
        opt = s["opt"]
        opt.step(lr, b1, b2, eps, wd, gscale=gscale)
        m, v, ms, vs, step = opt.m, opt.v, opt.m_scales, opt.v_scales, opt.step_dev
    else:
        step = s["step"].add_(1)
        n = s["g"].numel()
        g = s["g"].float() * gscale
        if c["bits"] == 8:
            m0 = (s["m"].float().view(-1, 128) / _power(s["m_scales"].to(torch.int32))[:, None]).view(-1)
            r0 = (s["v"].float().view(-1, 128) / _power(s["v_scales"].to(torch.int32))[:, None]).view(-1)
            v0 = r0 * r0
        else:
            m0, v0 = s["m"], s["v"]
        m1 = m0 * b1 + g * (1.0 - b1)
        v1 = v0 * b2 + (g * (1.0 - b2)) * g
        r1 = v1.sqrt()
        c1, c2 = (1.0 - b ** step.double() for b in (b1, b2))
        update = m1 / c1.float() / (r1 / c2.sqrt().float() + eps)
        w = s["master"] if s["master"] is not None else s["p"]
        w[:s["border"]] *= 1.0 - lr * wd
        w -= lr * update
        if s["master"] is not None:
            s["p"].copy_(w)
        if c["bits"] == 8:
            u = _random(n, s["seed"], step, w.device)
            for name, x, bits, positive in (("m", m1, u & 0xFFFF, False), ("v", r1, u >> 16, True)):
                q, e = _stochastic(x, bits, positive)
                s[name].copy_(q)
                s[name + "_scales"].copy_(e)
        else:
            m0.copy_(m1)
            v0.copy_(v1)
        m, v, ms, vs = s["m"], s["v"], s.get("m_scales"), s.get("v_scales")
    return {"p": s["p"], "master": s["master"], "m": m, "v": v, "m_scales": ms, "v_scales": vs, "step": step}


# ------------------------------------------------------------------ what cannot be done without
def work(case):
    if case["op"] == "quantize":
        n, copies = case["rows"] * case["cols"], 2 if case["both"] else 1
        return {"bytes": n * (TYPES[case["dtype"]].itemsize + copies * (1 + 1 / 128)), "flops": 0}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k * (1 + 1 / 128) + 2 * m * n + 2 * n * case["bias"] + m * k * (1 + 1 / 128) * case["keep"], "flops": 2 * m * n * k}
    if case["op"] == "backward":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * n + (n * k + m * k) * (1 + 1 / 128) + 2 * m * k + n * k * TYPES[case["dw"]].itemsize, "flops": 4 * m * n * k}
    n = sum(map(sum, _sizes(case)))
    return {"bytes": n * (TYPES[case["grad"]].itemsize + (10 if case["master"] else 8) + (16 if case["bits"] == 32 else 4 * (1 + 1 / 128))), "flops": 12 * n}


# ------------------------------------------------------------------ the same in 64 bits, from the definition
def _exact_scale(top):
    """The exponent s, at least -126, smallest with top <= 448 * 2^s"""
    f, e = torch.frexp(top)                       # 448 = 0.875 * 2^9
    s = e.double() - 9 + (f > 0.875)
    return torch.where(top > 0, s, -126.0).clamp(min=-126.0)


def _exact_steps(t):
    """The distance of e4m3's neighbours where t >= 0 lies"""
    return torch.exp2((torch.frexp(t)[1].double() - 1).clamp(min=-6.0) - 3)


def _exact_quantize(x, square=False, columns=False):
    """Along the rows of x (its columns: of x^T) in blocks of 128; what the matrix and q stand for"""
    x = (x.t() if columns else x).double()
    r, c = x.shape
    full = torch.nn.functional.pad(x, (0, -c % 128, 0, -r % 128))
    tiles = full.view(full.shape[0] // 128, 128, full.shape[1] // 128, 128)
    s = _exact_scale(tiles.abs().amax((1, 3) if square else 3))
    s = s[:, None, :, None] if square else s[..., None]
    t = tiles * torch.exp2(-s)
    step = _exact_steps(t.abs())
    q = torch.round(t / step) * step              # ties to even
    kp = full.shape[1]
    byte = (s.expand(tiles.shape[0], 128, kp // 128, 1).reshape(-1, kp // 128) + 127).to(torch.uint8)
    byte[r:] = 1
    return q.reshape(full.shape)[:r], byte, (q * torch.exp2(s)).reshape(full.shape)[:r, :c]


def _exact_out(q, byte):
    k = byte.shape[1]
    b = torch.ones(byte.shape[0], _up(k, 4) * 4, dtype=torch.uint8, device=byte.device)
    b[:, :k] = byte
    return [q, b.view(-1, 4, 32, b.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()]


def _exact_values(q):
    v, s = q
    e = s.permute(0, 3, 2, 1, 4).reshape(s.shape[0] * 128, -1)[:v.shape[0], :v.shape[1] // 128].double() - 127
    return v.double() * torch.exp2(e).repeat_interleave(128, 1)


def exact(case, seed):
    if case["op"] != "adamw":
        s = prepare(case, seed)
    if case["op"] == "quantize":
        q, b, _ = _exact_quantize(s["x"], case["square"])
        got = {"rows": _exact_out(q, b), "transposed": None}
        if case["both"]:
            q, b, _ = _exact_quantize(s["x"], case["square"], columns=True)
            got["transposed"] = _exact_out(q, b)
        return got
    if case["op"] == "linear":
        k = case["k"]
        y = _exact_quantize(s["x"])[2] @ _exact_values(s["w"])[:, :k].t()
        if s["bias"] is not None:
            y += s["bias"].double()
        return {"y": y, "keep": _exact_out(*_exact_quantize(s["x"], columns=True)[:2]) if case["keep"] else None}
    if case["op"] == "backward":
        m, n = case["m"], case["n"]
        dx = _exact_quantize(s["dy"])[2] @ _exact_values(s["wt"])[:, :n].t()
        dw = _exact_quantize(s["dy"], columns=True)[2] @ _exact_values(s["xt"])[:, :m].t()
        return {"dx": dx, "dw": dw}
    global own
    kept, own = own, False                        # the state as plain tensors
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return _exact_adamw(case, s)


def _exact_adamw(case, s):
    lr, b1, b2, eps, wd, gscale = s["rates"]
    t = case["step"] + 1
    g = s["g"].double() * gscale
    if case["bits"] == 8:
        m, r = ((s[a].double().view(-1, 128) * torch.exp2(s[a + "_scales"].double() - 127)[:, None]).view(-1) for a in ("m", "v"))
        v = r * r
    else:
        m, v = s["m"].double(), s["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    w = (s["p"] if s["master"] is None else s["master"]).double()
    keep = torch.ones_like(w)
    keep[:s["border"]] = 1 - lr * wd
    w = w * keep - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    out = {"p": w, "master": None if s["master"] is None else w, "m": m, "v": v, "m_scales": None, "v_scales": None, "step": s["step"] + 1}
    if case["bits"] == 8:
        mask = 0xFFFFFFFF
        h = (torch.arange(w.numel(), device=w.device) * 0x9E3779B9 + ((s["seed"] + t * 0x9E3779B9) & mask)) & mask
        h = ((h ^ (h >> 16)) * 0xBB67AE85) & mask
        h = ((h ^ (h >> 15)) * 0x6A09E667) & mask
        h ^= h >> 16
        for a, x, bits in (("m", m, h & 0xFFFF), ("v", v.sqrt(), h >> 16)):
            x = x.view(-1, 128)
            e = _exact_scale(x.abs().amax(1))
            y = x * torch.exp2(-e)[:, None]
            step = _exact_steps(y.abs())
            q = torch.floor(y.abs() / step + bits.view(-1, 128).double() / 65536) * step
            q = torch.where((q == 0) & (y != 0), 2.0 ** -9, q) if a == "v" else q
            out[a] = (q * torch.sign(y)).view(-1)
            out[a + "_scales"] = (e + 127).to(torch.uint8)
    return out
