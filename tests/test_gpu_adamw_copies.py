"""A copy of an optimiser steps its own parameters and moments."""

import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu


def saved(opt):
    f = io.BytesIO()
    torch.save(opt, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("copied", [copy.deepcopy, saved])
def test_copies(oztt, cuda, bits, copied):
    sizes = [300, 9001]
    def grads(t):
        g = torch.Generator(device="cuda").manual_seed(t)
        return [torch.randn(n, device="cuda", generator=g) for n in sizes]
    a = oztt.AdamW([torch.ones(n, device="cuda").bfloat16() for n in sizes], masters=True, state_bits=bits, seed=3)
    a.step(grads(1))
    b = copied(a)
    state = lambda o: [t.clone() for t in (*o.params, *o.masters, *o.moments())]  # noqa: E731
    kept = state(a)
    b.step(grads(2))
    after = state(b)
    assert all(torch.equal(x, y) for x, y in zip(kept, state(a)))  # the copy's step left the original alone
    assert not torch.equal(after[0], kept[0]) and b.t == 2 and a.t == 1
    a.step(grads(2))
    assert all(torch.equal(x, y) for x, y in zip(after, state(a)))
    del a
    torch.cuda.empty_cache()
    b.step(grads(3))
    assert bool(torch.isfinite(b.masters[0]).all())


def test_buffers_that_changed_are_refused(oztt, cuda):
    opt = oztt.AdamW([torch.ones(300, device="cuda")], state_bits=8)
    kept = opt._m
    for other in (kept.float(), kept[:256], kept.cpu(), torch.zeros(1024, dtype=torch.uint8, device="cuda")[::2], None):
        opt._m = other
        with pytest.raises(ValueError):
            opt.step([torch.ones(300, device="cuda")])
        with pytest.raises(ValueError):
            opt.moments()
    opt._m = kept
    opt.step([torch.ones(300, device="cuda")])
    assert opt.t == 1
