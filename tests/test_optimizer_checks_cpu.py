"""What AdamW over many tensors refuses (no GPU needed: nothing is launched)."""
from contextlib import contextmanager

import pytest
import torch


def test_a_capture_on_the_optimisers_own_device_counts(monkeypatch):
    """Gradients are exchanged by a copy on the current stream of the parameters' device, which need not be the current device."""
    from piccl_b200.ops import optimizer
    there = []

    @contextmanager
    def on(device):
        there.append(device)
        yield
        there.pop()

    monkeypatch.setattr(optimizer, "_on", on)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: there == [torch.device("cuda", 1)])
    opt = optimizer.AdamW.__new__(optimizer.AdamW)
    opt._device, opt._params = torch.device("cuda", 1), (torch.zeros(4),)
    with pytest.raises(RuntimeError, match="capture"):
        opt.set_grads([torch.zeros(4)])
