"""The layer operators under torch's forward mode: an error, never a result that lost its tangent."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu


def tensors(dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return r(40, 96), r(72, 96) / 8, r(72), r(40, 72)


def call(oztt, x, w, b, r):
    return oztt.linear(x, w, b, residual=r, activation="silu")


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_is_refused(oztt, cuda, which):
    t = list(tensors())
    with fwad.dual_level():
        t[which] = fwad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(oztt, *t)


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_through_the_gradients_is_refused(oztt, cuda, which):
    x, w, b, dy = tensors()
    t = [dy, x, w, dy.roll(1, 0)]
    with fwad.dual_level():
        t[which] = fwad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            oztt.linear_backward(*t[:3], pre=t[3], activation="silu")
