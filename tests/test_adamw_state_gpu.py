"""The moments of AdamW, step after step against their definition in plain single-precision operations, which never takes over what the kernel holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu


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
