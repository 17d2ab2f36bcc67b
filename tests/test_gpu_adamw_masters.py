"""FP32 parameters with FP32 masters: the step is taken on the master, and the parameter is the master."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_fp32_parameter_with_master(oztt, cuda, bits, grad, offset):
    """Three steps give the parameter, its master and a parameter without one the same values bit for bit, beside
    16-bit parameters with masters in the same call; nothing beside the parameter is written."""
    sizes = [1, 255, 256, 300, 9001]
    room = [torch.full((n + 16,), 7.0, device="cuda") for n in sizes]
    params = [r[4 + offset:4 + offset + n].copy_(torch.randn(n, device="cuda")) for r, n in zip(room, sizes)]
    alone = [p.clone() for p in params]
    halves = [p.bfloat16() for p in params]
    masters = [p.clone() for p in params]
    kw = dict(lr=3e-3, weight_decay=0.1, state_bits=bits, seed=5)
    a = oztt.AdamW(params + halves, masters=masters + [h.float() for h in halves], **kw)
    b = oztt.AdamW(alone + [h.clone() for h in halves], masters=[None] * len(sizes) + [h.float() for h in halves], **kw)
    start = [p.clone() for p in params]
    for t in range(3):
        grads = [torch.randn(n, device="cuda").to(grad) for n in sizes] * 2
        a.step(grads)
        b.step(grads)
        for p, w, q, s, n in zip(params, masters, alone, start, sizes):
            assert torch.equal(w, q) and not torch.equal(w, s)
            assert torch.equal(p, w)
        assert all(torch.equal(h, w.bfloat16()) for h, w in zip(halves, a.masters[len(sizes):]))
    for r, n in zip(room, sizes):
        assert bool((torch.cat([r[:4 + offset], r[4 + offset + n:]]) == 7.0).all())
