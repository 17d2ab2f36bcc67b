"""What the layer calls need beside their results comes from torch's allocator."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_scratch_is_torchs(oztt, cuda):
    """What a call needs beside its results comes from torch's allocator, on the call's stream: dz, and the copies of
    operands that do not start on 16 bytes."""
    m, n, k = 2048, 1024, 512
    x, w, dy = (torch.randn(*s, device="cuda").bfloat16() for s in ((m, k), (n, k), (m, n)))
    xo, wo = (torch.randn(s[0] * s[1] + 1, device="cuda").bfloat16()[1:].view(*s) for s in ((m, k), (n, k)))
    for call, results, scratch in (
            (lambda: oztt.linear_backward(dy, x, w, pre=dy, activation="relu"), 2 * (m * k + n * k + n), 2 * m * n),
            (lambda: oztt.linear(xo, wo), 2 * m * n, 2 * (m * k + n * k))):
        call()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = call()
        peak = torch.cuda.max_memory_allocated() - before
        assert results + scratch <= peak <= 1.1 * (results + scratch) + (1 << 20)
        del out


def test_out_of_memory_is_torchs(oztt, cuda):
    """Results too large for the card (a weight of one value repeated needs no memory itself)."""
    x = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(torch.OutOfMemoryError):
        oztt.linear(x.expand(1 << 20, 1), x.expand(1 << 20, 1))
    with pytest.raises(torch.OutOfMemoryError):  # dz alone
        y = x.expand(1 << 20, 1 << 20)
        oztt.linear_backward(y, x.expand(1 << 20, 1), x.expand(1 << 20, 1), pre=y, activation="relu", need_weight=False,
                             need_bias=False)
    assert float(oztt.linear(x, x)) == 0.0
