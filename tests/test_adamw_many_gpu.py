"""AdamW over many tensors against the formula in 64 bits, and its 8-bit moments against their definition in single roundings."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

RATES = dict(lr=1e-3, b1=0.9, b2=0.95, eps=1e-8, wd=0.1)
SIZES = [1, 2, 3, 4, 5, 127, 128, 129, 0, 131, 512, 1000, 4097, 70001]


def _tensors(sizes, master, grad, offset=0, seed=0, scale=1e-3):
    """(params, masters, grads): views that start `offset` elements into their buffers"""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(n, dtype, std):
        return (torch.randn(n + offset, generator=g, device="cuda") * std).to(dtype)[offset:]

    w = [t(n, torch.float32, 0.02) for n in sizes]
    size = [scale * math.exp(i % 5 - 2) for i in range(len(sizes))]
    grads = [t(n, grad, s) for n, s in zip(sizes, size)]
    if not master:
        return w, None, grads
    params = []
    for x in w:
        p = torch.empty(x.numel() + offset, dtype=torch.bfloat16, device="cuda")[offset:]
        p.copy_(x)
        params.append(p)
    return params, w, grads


def _reference(w, m, v, g, t, decay, gscale=1.0, lr=0.0, b1=0.0, b2=0.0, eps=0.0, wd=0.0):
    """The formula in fp64, and the size of what is taken off a weight as its roundings count it: the sum that gives m may cancel, its addends' roundings do not.  These are some 16 half steps of fp32:
    three of m, as many of each of 1 - b^t and its reciprocal, one of lr, two of an approximate root, one of eps, four of a quotient that is right to two steps."""
    g = g.double() * gscale
    size = lr * (b1 * m.double().abs() + (1 - b1) * g.abs()) / (1 - b1 ** t)
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g * g
    below = (v / (1 - b2 ** t)).sqrt() + eps
    return w.double() * (1 - lr * (wd if decay else 0.0)) - lr * (m / (1 - b1 ** t)) / below, m, v, size / below


def _near(got, want, old, steps, change):
    """got, rounded a few times to fp32: off by `steps` half steps of what it is computed from, and as much of the change"""
    bound = steps * 2.0 ** -24 * (old.double().abs() + want.abs() + change)
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound.clamp(min=1e-300)).max())


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("grad", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_moments_in_32_bits(master, grad, offset):
    from piccl_b200.ops.optimizer import AdamW
    params, masters, grads = _tensors(SIZES, master, grad, offset)
    decay = [i % 2 == 0 for i in range(len(SIZES))]
    opt = AdamW(params, grads, masters, decay=decay)
    weights = masters or params
    for step in range(1, 4):
        before = [(w.clone(), *opt.moments(i)) for i, w in enumerate(weights)]
        opt.step(gscale=0.7, **RATES)
        assert int(opt.step_dev) == step
        for i, (w, m, v) in enumerate(before):
            want = _reference(w, m, v, grads[i], step, decay[i], 0.7, **RATES)
            got = opt.moments(i)
            # m and v: two products and a sum, the gradient's scaling before
            _near(got[0], want[1], m, 4, grads[i].double().abs())
            _near(got[1], want[2], v, 6, (grads[i].double()) ** 2)
            _near(weights[i], want[0], w, 2, 10 * want[3])
            if master:
                assert torch.equal(params[i], weights[i].to(torch.bfloat16))


def _bytes(x):
    b = x.abs()
    top = torch.where(b.isfinite(), b, 0.0).amax(1)
    return (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=1)


def _bits(n, seed, step):
    mask = 0xFFFFFFFF
    h = (torch.arange(n, device="cuda") * 0x9E3779B9 + seed + step * 0x9E3779B9) & mask
    h = ((h ^ (h >> 16)) * 0xBB67AE85) & mask
    h = ((h ^ (h >> 15)) * 0x6A09E667) & mask
    return h ^ (h >> 16)


def _held(x, u, positive, off=0.0):
    """(e4m3 values, bytes) of blocks, stochastically rounded, in fp64 from what fp32 arithmetic gave (times 1 + off)"""
    byte = _bytes(x)
    t = (x.double() * torch.exp2(127.0 - byte.double())[:, None] * (1 + off)).clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
    q = torch.floor(t.abs() / step + u.double() / 65536) * step
    if positive:
        q = torch.where((q == 0) & (t != 0), 2.0 ** -9, q)
    return torch.where(x.isfinite(), torch.copysign(q, t), math.nan), byte


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("grad", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1])
def test_moments_in_8_bits(master, grad, offset):
    from piccl_b200.ops.optimizer import AdamW
    params, masters, grads = _tensors(SIZES, master, grad, offset, seed=3)
    if grad == torch.float32:
        grads[-1][::7] *= 2.0 ** -14                    # far below the largest of their block
    grads[-2][:256] = 0
    seed = 12345
    opt = AdamW(params, grads, masters, bits=8, seed=seed)
    weights = masters or params
    f = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    for step in range(1, 5):
        before = [(w.clone(), *opt.moments(i)) for i, w in enumerate(weights)]
        u = _bits(opt.blocks * 128, seed, step)
        opt.step(gscale=0.7, **RATES)
        for i, (w, m, v) in enumerate(before):
            n, o = w.numel(), opt.places[i][0]
            if n == 0:
                continue
            x = grads[i].float() * f(0.7)
            m1 = m * f(0.9) + x * f(1 - 0.9)
            v1 = v * f(0.95) + (x * f(1 - 0.95)) * x
            blocks = (n + 127) // 128
            for held, scales, now, r, positive in ((opt.m, opt.m_scales, m1, u & 0xFFFF, False), (opt.v, opt.v_scales, v1.sqrt(), u >> 16, True)):
                full = torch.zeros(blocks * 128, device="cuda")
                full[:n] = now
                q, byte = _held(full.view(blocks, 128), r[o:o + blocks * 128].view(blocks, 128), positive)
                assert torch.equal(scales[o // 128:o // 128 + blocks].int(), byte)
                got, same = held[o:o + blocks * 128].double(), False
                if positive:                        # the root is approximate, to 2^-22 of its value: it may be held as its neighbour within that would be
                    for off in (-2.0 ** -22, 2.0 ** -22):
                        same |= got == _held(full.view(blocks, 128), r[o:o + blocks * 128].view(blocks, 128), positive, off)[0].view(-1)
                same |= got == q.view(-1)
                assert bool(same.all())
            want = _reference(w, m, v, grads[i], step, True, 0.7, **RATES)
            _near(weights[i], want[0], w, 2, 10 * want[3])
            if master:
                assert torch.equal(params[i], weights[i].to(torch.bfloat16))


def test_values_that_are_not_finite_stay_in_their_place():
    from piccl_b200.ops.optimizer import AdamW
    for bits in (8, 32):
        params, _, grads = _tensors([300], False, torch.float32)
        grads[0][5], grads[0][200] = math.nan, math.inf
        opt = AdamW(params, grads, bits=bits)
        opt.step(**RATES)
        bad = torch.zeros(300, dtype=torch.bool, device="cuda")
        bad[5] = bad[200] = True
        assert torch.equal(~params[0].isfinite(), bad)
        m, v = opt.moments(0)
        assert torch.equal(~m.isfinite(), bad) and torch.equal(~v.isfinite(), bad)


def test_rounding_has_no_bias_and_nothing_stands_still():
    """A constant gradient with b2 = 0.999 after one of another size: nearest rounding would leave the root where it is (0.05 % a step, half a step of e4m3 is 3 %).  The mean of n
    independent roots has a deviation of at most s / sqrt(n), s the deviation of one; eight of them are allowed, s from the sample itself."""
    from piccl_b200.ops.optimizer import AdamW
    n = 1 << 16
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 1e-3, device="cuda")
    opt = AdamW([p], [g], bits=8)
    rates = dict(lr=0.0, b1=0.9, b2=0.999, eps=1e-8, wd=0.0)
    for _ in range(20):
        opt.step(**rates)
    g.fill_(1e-4)
    root = opt.moments(0)[1].sqrt().double()
    for _ in range(20):
        before = root.mean()
        exact = (0.999 * root ** 2 + 0.001 * 1e-8).sqrt().mean()           # of what is held, before it is rounded again
        opt.step(**rates)
        root = opt.moments(0)[1].sqrt().double()
        assert exact < before
        assert abs(root.mean() - exact) <= 8 * root.std() / math.sqrt(n) + 1e-12
    m = opt.moments(0)[0].double()
    expected = 1e-4 + (1e-3 * (1 - 0.9 ** 20) - 1e-4) * 0.9 ** 20
    assert abs(m.mean() - expected) <= 8 * m.std() / math.sqrt(n) + 1e-6 * expected


def test_step_in_a_graph_and_a_device_factor():
    """Replays go on counting, and draw other bits: the state is that of as many steps issued one by one."""
    from piccl_b200.ops.optimizer import AdamW
    for bits in (8, 32):
        runs = []
        for captured in (False, True):
            params, masters, grads = _tensors(SIZES, True, torch.bfloat16, seed=9)
            factor = torch.full((1,), 0.5, device="cuda")
            opt = AdamW(params, grads, masters, bits=bits, seed=7)
            opt.step(gscale=factor, **RATES)
            if captured:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    opt.step(gscale=factor, **RATES)
                step = graph.replay
            else:
                step = lambda: opt.step(gscale=factor, **RATES)  # noqa: E731
            for k in range(3):
                factor.fill_(0.25 * (k + 1))
                step()
            assert int(opt.step_dev) == 4
            runs.append([*params, *masters, opt.m.float(), opt.v.float(), *([opt.m_scales, opt.v_scales] if bits == 8 else [])])
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_more_tensors_than_blocks_and_other_gradients():
    from piccl_b200.ops.optimizer import AdamW
    sizes = [1 + i % 3 for i in range(3000)]
    params, _, grads = _tensors(sizes, False, torch.float32, seed=1)
    opt = AdamW(params, grads)
    before = [w.clone() for w in params]
    others = [g * 2 for g in grads]
    opt.set_grads(others)
    opt.step(**RATES)
    w0, g0 = torch.cat(before), torch.cat(others)
    want = _reference(w0, torch.zeros_like(w0), torch.zeros_like(w0), g0, 1, True, **RATES)
    _near(torch.cat(params), want[0], w0, 2, 10 * want[3])


def test_gpt2_with_moments_in_8_bits():
    """The first step is that of moments in 32 bits (nothing has been rounded before it), and replayed steps of the trainer are those issued one by one."""
    from piccl_b200.models.gpt2 import GPT2, GPT2Config
    from piccl_b200.train import DataParallelTrainer
    cfg = GPT2Config.tiny()
    tok = torch.randint(0, cfg.vocab_size, (2, cfg.seq_len + 1), generator=torch.Generator().manual_seed(0))
    a, b = tok[:, :-1].contiguous(), tok[:, 1:].contiguous()
    models = [GPT2(cfg, seed=3, adam_bits=bits) for bits in (32, 8)]
    for m in models:
        m.forward_backward(a.cuda(), b.cuda())
    assert torch.equal(models[0].flat_g, models[1].flat_g)
    before = models[0].master.clone()
    for m in models:
        m.optimizer_step(lr=1e-3)
    w32, w8 = (m.master.double() for m in models)
    _near(models[1].master, w32, before, 4, 20 * (w32 - before.double()).abs())
    assert torch.equal(models[1].flat_p, models[1].master.to(torch.bfloat16)) and int(models[1].step_dev) == 1
    runs = []
    for graph in (False, True):
        tr = DataParallelTrainer(cfg, None, seed=3, adam_bits=8, use_graph=graph)
        losses = [tr.step(a.pin_memory(), b.pin_memory()) for _ in range(5)]
        assert int(tr.model.step_dev) == tr.model.step_count == 5
        runs.append((losses, tr.model.master.clone(), tr.model.m.float()))
    assert all(math.isfinite(x) for x in runs[0][0] + runs[1][0])
    with pytest.raises(ValueError):
        GPT2(cfg, adam_bits=16)


def test_gradients_beside_their_parameters_in_a_buffer():
    """Next to each other is fine, overlapping is refused: other lanes would read what one has written."""
    from piccl_b200.ops.optimizer import AdamW
    buf = torch.ones(64, device="cuda")
    opt = AdamW([buf[16:32], buf[40:48]], [buf[0:16], buf[32:40]])
    opt.set_grads([buf[48:64], buf[8:16]])
    for grads in ([buf[16:32], buf[32:40]], [buf[8:24], buf[32:40]], [buf[24:40], buf[32:40]], [buf[0:16], buf[47:55]], [buf[0:16], buf[33:41]], [torch.zeros(16, device="cuda"), buf.view(torch.bfloat16)[94:102]]):
        with pytest.raises(ValueError, match="overlap"):
            opt.set_grads(grads)
    opt.step(0.0, wd=0.0)
    assert bool((buf == 1).all()) and torch.equal(opt.moments(0)[0], torch.full((16,), torch.tensor(1 - 0.9, dtype=torch.float32).item(), device="cuda"))


def test_refusals_on_the_gpu():
    from piccl_b200.ops.optimizer import AdamW
    p, g = torch.ones(16, device="cuda"), torch.ones(16, device="cuda")
    opt = AdamW([p], [g])
    for kw in (dict(b1=1.0), dict(b2=-0.5), dict(gscale=torch.ones(2, device="cuda")), dict(gscale=torch.ones(1)), dict(gscale=torch.ones(1, device="cuda", dtype=torch.float64))):
        with pytest.raises(ValueError):
            opt.step(1e-3, **kw)
    for grads in ([], [g[:8]], [g.double()], [g.cpu()], [torch.ones(32, device="cuda")[::2]]):
        with pytest.raises(ValueError):
            opt.set_grads(grads)
    for params in ([p, p], [p, p[8:]], [p[:9], p[8:]]):
        with pytest.raises(ValueError, match="overlap"):
            AdamW(params, [torch.zeros_like(t) for t in params])
    assert int(opt.step_dev) == 0 and bool((p == 1).all())
    graph = torch.cuda.CUDAGraph()
    opt.step(0.0, wd=0.0)
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            opt.set_grads([g])
        opt.step(0.0, wd=0.0)
    none = AdamW([torch.empty(0, device="cuda")], [torch.empty(0, device="cuda")], bits=8)
    none.step(1e-3)
    assert int(none.step_dev) == 1
