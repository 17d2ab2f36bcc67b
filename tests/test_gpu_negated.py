"""Lazily negated tensors, whose memory holds the negative of what they stand for."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def tensors(dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return r(40, 96), r(72, 96) / 8, r(72), r(40, 72)


def call(oztt, x, w, b, r):
    return oztt.linear(x, w, b, residual=r, activation="silu")


def test_lazily_negated(oztt, cuda):
    """x.imag of a conjugate is a view that stands for the negative of what lies in memory."""
    x, w, b, r = tensors(torch.float16)
    def negated(t):
        n = torch.view_as_complex(torch.stack([t, -t], -1).contiguous()).conj().imag
        assert n.is_neg() and torch.equal(n.clone(), t)
        return n
    for i in range(4):
        t = [x, w, b, r]
        want = call(oztt, *t)
        t[i] = negated(t[i])
        assert torch.equal(call(oztt, *t), want)
    pre = r.roll(1, 0)
    want = oztt.linear_backward(r, x, w, pre=pre, activation="gelu")
    for i in range(4):
        t = [r, x, w, pre]
        t[i] = negated(t[i])
        got = oztt.linear_backward(*t[:3], pre=t[3], activation="gelu")
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_zeros_without_memory(oztt, cuda):
    """torch's derivatives give zeros that have no memory."""
    x, w, b, r = tensors()
    zero = torch._efficientzerotensor(r.shape, dtype=r.dtype, device="cuda")
    assert torch.equal(oztt.linear(x, w, b, residual=zero), oztt.linear(x, w, b))
    dx, dw, db = oztt.linear_backward(zero, x, w)
    assert not bool(dx.any()) and not bool(dw.any()) and not bool(db.any())
