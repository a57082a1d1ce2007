"""The moments of AdamW, step after step against their definition in plain single-precision operations, which never takes over what the kernel holds."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24          # half a step of fp32, relative to the value


def _random(n, seed, step):
    """The definition's 32 random bits for each place"""
    mask = 0xFFFFFFFF
    h = torch.arange(n, device="cuda").mul_(0x9E3779B9).add_(seed + step * 0x9E3779B9).bitwise_and_(mask)
    h = ((h ^ (h >> 16)) * 0xBB67AE85) & mask
    h = ((h ^ (h >> 15)) * 0x6A09E667) & mask
    return h ^ (h >> 16)


def _hold(x, u, positive):
    """fp32 values of whole blocks of 128 -> what the bytes stand for (before the scale) and the scales' bytes: rounded up with the probability of the part cut off"""
    b = x.view(-1, 128)
    top = torch.where(b.isfinite(), b.abs(), 0.0).amax(1)
    byte = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=1)
    t = b * ((254 - byte) << 23).view(torch.float32)[:, None]
    a = t.abs()
    low = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)          # below, e4m3's steps are those of [2^-6, 2^-5)
    z = (a + low).view(torch.int32) + (u.view(-1, 128) << 4).to(torch.int32)
    z = (z & ~0xFFFFF).view(torch.float32) - low
    if positive:
        z = torch.where(a > 0, z.clamp(min=2.0 ** -9), z)
    return z.copysign(t).view(-1), byte


def _value(z, byte):
    return (z.view(-1, 128) * (byte << 23).view(torch.float32)[:, None]).view(-1)


class _Plain:
    """The state as fp32 tensors of whole blocks; the weights follow it in fp64, with a bound on what fp32 may lose from them"""

    def __init__(self, w):
        n = w.numel()
        full = (n + 127) // 128 * 128
        self.n, self.w, self.allowed = n, w.double(), torch.zeros(n, dtype=torch.float64, device="cuda")
        self.zm, self.zr = torch.zeros(full, device="cuda"), torch.zeros(full, device="cuda")
        self.em, self.er = (torch.ones(full // 128, dtype=torch.int32, device="cuda") for _ in range(2))
        self.t = 0

    def step(self, g, seed, lr, b1, b2, eps, wd, gscale):
        self.t += 1
        x = torch.zeros_like(self.zm)
        x[:self.n] = g.float() * gscale
        m, r = _value(self.zm, self.em), _value(self.zr, self.er)
        m = m * b1 + x * (1.0 - b1)
        v = (r * r) * b2 + (x * (1.0 - b2)) * x
        u = _random(x.numel(), seed, self.t)
        self.zm, self.em = _hold(m, u & 0xFFFF, False)
        self.zr, self.er = _hold(v.sqrt(), u >> 16, True)
        m, v = m[:self.n].double(), v[:self.n].double()
        change = lr * (m / (1 - b1 ** self.t)) / ((v / (1 - b2 ** self.t)).sqrt() + eps)
        after = self.w * (1 - lr * wd) - change
        # 13 half steps of the change: three of each of 1 - b^t and its reciprocal, one of lr, two of an approximate root, one of eps, four of a quotient that is right to two steps (and 20 stand here); one of
        # the factor of the weight, one of the result
        self.allowed += 2 * HALF * (self.w.abs() + after.abs() + 10 * change.abs())
        self.w = after


def _compare(opt, plain, p):
    assert torch.equal(opt.m_scales.int(), plain.em) and torch.equal(opt.v_scales.int(), plain.er)
    assert torch.equal(opt.m.float(), plain.zm), int((opt.m.float() != plain.zm).sum())
    assert torch.equal(opt.v.float(), plain.zr), int((opt.v.float() != plain.zr).sum())
    off = (p.double() - plain.w).abs()
    assert bool((off <= plain.allowed).all()), float((off / plain.allowed.clamp(min=1e-300)).max())


def test_eight_steps_side_by_side():
    """The state is the definition's bit for bit, with the correctly rounded root (one unit in the last place moves a held root by a whole step of e4m3 where it tips the carry, in an element
    of 10^6 a step, and the next step divides by that), and so the weights stay where sums in fp32 put them."""
    from piccl_b200.ops.optimizer import AdamW
    n, seed = (1 << 25) + 77, 21
    gen = torch.Generator(device="cuda").manual_seed(5)
    size = torch.exp(torch.randn(n // 128 + 1, 1, generator=gen, device="cuda") - 9.0).expand(-1, 128).reshape(-1)[:n]
    w = torch.randn(n, generator=gen, device="cuda") * 0.02
    p, g = w.clone(), torch.empty(n, dtype=torch.bfloat16, device="cuda")
    opt, plain = AdamW([p], [g], bits=8, seed=seed), _Plain(w)
    del w
    for _ in range(8):
        g.copy_(torch.randn(n, generator=gen, device="cuda") * size)
        g[1 << 20:(1 << 20) + 500] = 0
        opt.step(3e-4, 0.9, 0.95, 1e-8, 0.1, gscale=0.7)
        plain.step(g, seed, 3e-4, 0.9, 0.95, 1e-8, 0.1, 0.7)
        _compare(opt, plain, p)


@pytest.mark.parametrize("eps", [0.0, 1e-8])
@pytest.mark.parametrize("size", [2.0 ** -62, 2.0 ** -66, 2.0 ** -70])
def test_second_moments_below_the_normal_numbers(size, eps):
    """v is below 2^-126, its root a normal number: no root that is not zero becomes zero, and the update divides by it."""
    from piccl_b200.ops.optimizer import AdamW
    n, seed = 128 * 300 + 5, 3
    gen = torch.Generator(device="cuda").manual_seed(9)
    w = torch.randn(n, generator=gen, device="cuda")
    p, g = w.clone(), torch.zeros(n, device="cuda")
    opt, plain = AdamW([p], [g], bits=8, seed=seed), _Plain(w)
    for _ in range(3):
        g.copy_((torch.rand(n, generator=gen, device="cuda") + 0.5) * torch.randn(n, generator=gen, device="cuda").sign() * size)
        if eps:
            g[128:256] = 0          # nothing there
            g[260:300] *= 2.0 ** 40          # beside values far above
        opt.step(1e-3, 0.9, 0.95, eps, 0.1)
        plain.step(g, seed, 1e-3, 0.9, 0.95, eps, 0.1, 1.0)
        assert bool((opt.v.float()[:n][g != 0] > 0).all())
        _compare(opt, plain, p)


def test_the_largest_gradients():
    """Second moments up to fp32's largest."""
    from piccl_b200.ops.optimizer import AdamW
    n, seed = 128 * 40 + 3, 4
    gen = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(n, generator=gen, device="cuda")
    p, g = w.clone(), torch.zeros(n, device="cuda")
    opt, plain = AdamW([p], [g], bits=8, seed=seed), _Plain(w)
    for _ in range(3):
        g.copy_(torch.randn(n, generator=gen, device="cuda").clamp(-4, 4) * 4.0e18)
        opt.step(1e-3, 0.9, 0.95, 1e-8, 0.1)
        plain.step(g, seed, 1e-3, 0.9, 0.95, 1e-8, 0.1, 1.0)
        _compare(opt, plain, p)
    assert math.isfinite(float(p.abs().max()))


def test_moments_in_32_bits_are_rounded_one_operation_at_a_time():
    """Products and their sum are rounded each by itself, as plain operations do it; fused, a quarter of the moments would be off by their last bit (and held otherwise in 8 bits)."""
    from piccl_b200.ops.optimizer import AdamW
    n = (1 << 20) + 5
    gen = torch.Generator(device="cuda").manual_seed(5)
    w, g = torch.randn(n, generator=gen, device="cuda"), torch.randn(n, generator=gen, device="cuda")
    for buffers in ((w, g), (w[1:], g[1:])):          # words, and element by element
        opt = AdamW([buffers[0]], [buffers[1]])
        opt.m.copy_(torch.randn(opt.m.numel(), generator=gen, device="cuda"))
        opt.v.copy_(torch.rand(opt.v.numel(), generator=gen, device="cuda"))
        m, v = opt.moments(0)
        x = buffers[1] * 0.7
        opt.step(1e-3, 0.9, 0.95, 1e-8, 0.1, gscale=0.7)
        got = opt.moments(0)
        assert torch.equal(got[0], m * 0.9 + x * (1.0 - 0.9)) and torch.equal(got[1], v * 0.95 + (x * (1.0 - 0.95)) * x)


@pytest.fixture(params=["native", "ctypes"])
def path(request, monkeypatch):
    """Each call path in turn (ctypes: as where Python's headers are missing)"""
    from piccl_b200.ops import fp8
    if request.param == "ctypes":
        monkeypatch.setattr(fp8, "_fast", False)
    else:
        assert fp8._native_calls()
    return request.param


@pytest.mark.parametrize("bits", [8, 32])
def test_the_state_cannot_part_from_the_steps(path, bits):
    """Captured steps and the native handle have the addresses: another tensor in the place of one of these would be passed over, and what it replaced freed under the next step."""
    from piccl_b200.ops.optimizer import AdamW
    p, g = torch.ones(300, device="cuda"), torch.full((300,), 1e-3, device="cuda")
    opt = AdamW([p], [g], bits=bits, seed=3)
    opt.step(1e-3)
    for name in ("m", "v", "m_scales", "v_scales", "step_dev", "seed", "bits", "params", "masters", "grads", "decay", "places", "blocks", "device"):
        kept = getattr(opt, name)
        with pytest.raises(AttributeError):
            setattr(opt, name, kept.clone() if isinstance(kept, torch.Tensor) else kept)
        assert getattr(opt, name) is kept or name == "seed"
    for name in ("params", "masters", "grads", "decay", "places"):
        assert isinstance(getattr(opt, name), tuple)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("where", ["cuda", "cpu"])
def test_a_state_is_loaded_in_place(path, bits, where):
    """An optimiser that goes on from another's state does what that one does, captured steps of its own among them."""
    from piccl_b200.ops.optimizer import AdamW
    sizes = [300, 0, 5, 4097]
    gen = torch.Generator(device="cuda").manual_seed(1)
    start = [torch.randn(n, generator=gen, device="cuda") for n in sizes]
    grads = [torch.randn(n, generator=gen, device="cuda") * 1e-3 for n in sizes]

    def make():
        params = [w.clone() for w in start]
        return params, AdamW(params, grads, bits=bits, seed=7)

    a, one = make()
    for _ in range(3):
        one.step(1e-3)
    b, two = make()
    graph = torch.cuda.CUDAGraph()
    two.step(1e-3)
    with torch.cuda.graph(graph):
        two.step(1e-3)
    with torch.no_grad():
        for x, y in zip(a, b):
            y.copy_(x)
    two.load_state({k: t.to(where, copy=True) for k, t in one.state().items()})
    one.step(1e-3)
    graph.replay()
    one.step(1e-3)
    two.step(1e-3)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and int(two.step_dev) == 5
    assert all(torch.equal(t.float(), two.state()[k].float()) for k, t in one.state().items())
    for bad in ({}, {**one.state(), "m": one.m[:128]}, {**one.state(), "v": one.v.double()}, AdamW([torch.ones(300, device="cuda")], [grads[0]], bits=40 - bits).state()):
        with pytest.raises(ValueError):
            two.load_state(bad)


def test_tensors_that_have_moved_are_refused(path):
    """A step would write where a parameter was before it was given other memory, which may be another tensor's by now."""
    from piccl_b200.ops.optimizer import AdamW
    def make():
        w, p, g = torch.ones(300, device="cuda"), torch.ones(300, dtype=torch.bfloat16, device="cuda"), torch.ones(300, dtype=torch.bfloat16, device="cuda")
        return [w, p, g], AdamW([p], [g], [w])
    for i in range(3):
        tensors, opt = make()
        opt.step(1e-3)
        old = tensors[i].data
        tensors[i].data = tensors[i].data.clone()
        with pytest.raises(ValueError, match="not where it was"):
            opt.step(1e-3)
        if i < 2:
            with pytest.raises(ValueError, match="not where it was"):
                opt.set_grads([tensors[2]])
        else:
            opt.set_grads([tensors[2]])
            opt.step(1e-3)
        tensors[i].data = old
        if i == 2:
            opt.set_grads([tensors[2]])
        opt.step(1e-3)
        assert int(opt.step_dev) == (3 if i == 2 else 2)
        tensors[i].untyped_storage().resize_(0)
        with pytest.raises((ValueError, RuntimeError)):
            opt.step(1e-3)


def test_gpt2_says_that_its_state_stays_where_it_is():
    from piccl_b200.models.gpt2 import GPT2, GPT2Config
    model = GPT2(GPT2Config.tiny(), adam_bits=8)
    for name in ("master", "m", "v", "step_dev"):
        with pytest.raises(AttributeError):
            setattr(model, name, getattr(model, name).clone())
    assert model.m is model._adam.m and model.v is model._adam.v and model.step_dev is model._adam.step_dev
    model = GPT2(GPT2Config.tiny())          # with moments in 32 bits each step takes what is there
    for name in ("master", "m", "v", "step_dev"):
        other = getattr(model, name).clone()
        setattr(model, name, other)
        assert getattr(model, name) is other


@pytest.mark.parametrize("bits", [8, 32])
def test_replayed_steps_of_the_trainer_are_those_issued_one_by_one(bits):
    """Losses, weights and the optimiser's state, bit for bit: a replay goes on counting and draws other random bits than the capture."""
    from piccl_b200.models.gpt2 import GPT2Config
    from piccl_b200.train import DataParallelTrainer
    cfg = GPT2Config.tiny()
    tok = torch.randint(0, cfg.vocab_size, (6, 2, cfg.seq_len + 1), generator=torch.Generator().manual_seed(0))
    runs = []
    for graph in (False, True):
        tr = DataParallelTrainer(cfg, None, seed=3, adam_bits=bits, use_graph=graph)
        losses = [tr.step(t[:, :-1].contiguous().pin_memory(), t[:, 1:].contiguous().pin_memory()) for t in tok]
        state = tr.model._adam.state() if bits == 8 else {"m": tr.model.m, "v": tr.model.v, "step_dev": tr.model.step_dev}
        assert tr.replayed_steps() >= 3 if graph else True
        runs.append((losses, {"master": tr.model.master, "p": tr.model.flat_p, **state}))
    assert runs[0][0] == runs[1][0]
    for name, t in runs[0][1].items():
        assert torch.equal(t.float(), runs[1][1][name].float()), name


@pytest.mark.parametrize("b2,steps", [(0.95, 1000), (0.99, 2000), (0.999, 4000)])
def test_how_far_second_moments_in_8_bits_are_too_large(b2, steps):
    """The root is rounded without bias, so its square is too large by the rounding's variance.  A root r that would move by d is rounded up with the probability d / s of its step s, a variance of at most |d| s, with
    |d| <= (1 - b2) |g^2 - r^2| / (r (1 + sqrt b2)) and s <= r / 8.  In the mean V of the squares, k = 1 / (8 (1 + sqrt b2)): V <= b2 V + (1 - b2) (G + k (G + V)), so G <= V <= G (1 + k) / (1 - k), at any step.
    Of n elements the mean is off by no more than eight of its deviations, counted as if 2 / (1 - b2) neighbours went together, the steps that a moment remembers (a place's bits at a step are those of the place after it at
    the step before)."""
    from piccl_b200.ops.optimizer import AdamW
    n = 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(11)
    g = torch.empty(n, device="cuda")
    eight, full = (AdamW([torch.zeros(n, device="cuda")], [g], bits=bits, seed=1) for bits in (8, 32))
    for _ in range(steps):
        g.normal_(generator=gen)
        for o in (eight, full):
            o.step(0.0, 0.9, b2, 1e-8, 0.0)
    (m8, v8), (m32, v32) = (tuple(t.double() for t in o.moments(0)) for o in (eight, full))
    k, far = 1 / (8 * (1 + math.sqrt(b2))), 8 / math.sqrt(n * (1 - b2) / 2)
    ratio, spread = float(v8.mean() / v32.mean()), float((v8 / v32).std())
    print("mean", ratio, "deviation of one", spread)
    assert 1 - far * spread <= ratio <= (1 + k) / (1 - k) + far * spread
    # the first moment has no bias: its mean is that of the exact one within the same count
    assert abs(float((m8 - m32).mean())) <= 8 / math.sqrt(n * 0.1 / 2) * float((m8 - m32).std())


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("factor", [math.inf, math.nan])
def test_what_lies_between_tensors_stays_zero(bits, factor):
    """Also where the factor of the gradients is not finite, which makes NaN of every moment that is a tensor's: moments loaded over them are whole again, and a norm over the flat state is the tensors'."""
    from piccl_b200.ops.optimizer import AdamW
    sizes = [1, 130, 7, 256, 1001]
    params, grads = [torch.ones(n, device="cuda") for n in sizes], [torch.full((n,), 1e-3, device="cuda") for n in sizes]
    opt = AdamW(params, grads, bits=bits)
    opt.step(1e-3)
    opt.step(1e-3, gscale=torch.full((1,), factor, device="cuda"))
    inside = torch.zeros(opt.m.numel(), dtype=torch.bool, device="cuda")
    for o, n in opt.places:
        inside[o:o + n] = True
    for t in (opt.m.float(), opt.v.float()):
        assert bool((t[~inside] == 0).all()) and not bool(t[inside].isfinite().any())
