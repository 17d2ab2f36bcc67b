"""The optimiser where its writes would be missed."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu


def test_optimiser_refuses_what_it_would_miss(oztt, cuda):
    p = torch.ones(1, device="cuda")
    opt = oztt.AdamW([p], state_bits=8)
    negative = torch.view_as_complex(torch.ones(1, 2, device="cuda")).conj().imag
    assert negative.is_neg() and negative.is_contiguous()
    with pytest.raises(ValueError):
        opt.step([negative])
    with pytest.raises(ValueError):
        oztt.AdamW([negative])

    def stepped(g):
        opt.step([g])
        return p * 1

    for record in (lambda: torch.jit.trace(stepped, (torch.ones_like(p),), check_trace=False),
                   lambda: make_fx(stepped)(torch.ones_like(p)),
                   lambda: make_fx(lambda g: opt.moments()[0] + g)(torch.ones_like(p))):
        with pytest.raises((RuntimeError, ValueError)):
            record()
    assert opt.t == 0 and torch.equal(p, torch.ones_like(p))


def test_tensors_without_memory(oztt, cuda):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode() as mode:
        fake = mode.from_tensor(torch.zeros(10, device="cuda"))
    p = torch.zeros(10, device="cuda")
    with pytest.raises(ValueError):
        oztt.AdamW([fake])
    with pytest.raises(ValueError):
        oztt.AdamW([p], masters=[fake])
    with pytest.raises(ValueError):
        oztt.AdamW([p]).step([fake])
    opt, g = oztt.AdamW([p]), p + 1
    with FakeTensorMode(), pytest.raises(RuntimeError):
        opt.step([g])
    assert not bool(p.any())
