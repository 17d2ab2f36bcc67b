"""Offsets past 32 bits: outputs, operands and optimiser states of more than 2^31 elements. The last rows are compared
with the definition in 64 bits, and with the same rows computed by themselves."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_forward_past_32_bits(oztt, cuda):
    """2.2e9 outputs from operands of ordinary size, and x of 2.2e9 elements."""
    for m, n, k in ((140001, 16000, 64), (35000, 72, 64000)):
        x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16)
        w = torch.randn(n, k, device="cuda", dtype=torch.bfloat16)
        y = oztt.linear(x, w)
        rows = torch.tensor([0, 1, m // 2, m - 2, m - 1], device="cuda")
        want = x[rows].double() @ w.double().t()
        mag = x[rows].double().abs() @ w.double().abs().t()
        assert bool(((y[rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + (k + 2) * 2.0 ** -23 * mag).all())
        del x, w, y
        torch.cuda.empty_cache()


def test_backward_past_32_bits(oztt, cuda):
    """dz of 2.2e9 elements (a scratch matrix) and its sums."""
    m, n, k = 140001, 16000, 64
    x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(n, k, device="cuda", dtype=torch.bfloat16)
    dy = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    dy[-3:] = torch.randn(3, n, device="cuda")
    pre = torch.ones_like(dy)  # RELU passes everything
    dx, dw, db = oztt.linear_backward(dy, x, w, pre=pre, activation="relu")
    d = dy[-3:].double()
    want, mag = d @ w.double(), d.abs() @ w.double().abs()
    assert bool(((dx[-3:].double() - want).abs() <= 2.0 ** -8 * want.abs() + (n + 2) * 2.0 ** -23 * mag).all())
    assert not bool(dx[:-3].any())
    want, mag = d.t() @ x[-3:].double(), d.t().abs() @ x[-3:].double().abs()
    assert bool(((dw.double() - want).abs() <= 2.0 ** -8 * want.abs() + (m + 2) * 2.0 ** -23 * mag).all())
    want = d.sum(0)
    assert bool(((db.double() - want).abs() <= 2.0 ** -8 * want.abs() + (m + 2) * 2.0 ** -24 * d.abs().sum(0)).all())


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_past_32_bits(oztt, cuda, bits):
    """One tensor of 2.2e9 elements and one behind it, whose moments start past 2^31: the last stretch of the first
    and the second are what small tensors with the same values give (with 8 bits: to the spacing of a code, since
    the random numbers are those of their place)."""
    n, tail = 2_200_000_000, 256 * 40
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(tail, device="cuda").to(torch.bfloat16)
    p[-tail:] = q
    g = torch.zeros_like(p)
    g[-tail:] = torch.randn(tail, device="cuda")
    second = q.clone()
    opt = oztt.AdamW([p, second], state_bits=bits, weight_decay=0.1)
    small = oztt.AdamW([q], state_bits=bits, weight_decay=0.1)
    opt.step([g, g[-tail:].clone()])
    small.step([g[-tail:].clone()])
    assert torch.equal(p[-tail:], q) and torch.equal(second, q) and not bool(p[:-tail].any())
    (m, v), (sm, sv) = opt.moments(), small.moments()
    for flat, want in ((m, sm), (v, sv)):
        for at in (n - tail, opt.offsets[1]):
            got = flat[at:at + tail].float()
            if bits == 32:
                assert torch.equal(got, want)
            else:  # neighbouring codes: at most 1/8 apart, or the smallest code of a block
                assert bool(((got - want.float()).abs() <= want.float().abs() / 8 + 2.0 ** -14 * want.float().abs().max()).all())
    assert opt.offsets[1] > 2 ** 31 and not bool(m[:n - tail].any())
