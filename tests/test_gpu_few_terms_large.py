"""Gradients of 6 to 8 tokens on both sides of the size from which tiles form them, against 64 bits: each product of two
16-bit values is exact in 32 bits and m of them are summed (m 2^-23 of the magnitudes), then rounded once."""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [6, 7, 8])
@pytest.mark.parametrize("n,k", [(5000, 7992), (5000, 8000), (4999, 8008), (16, 2500008)])
def test_dw(oztt, cuda, dtype, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m)
    x, dy = (torch.randn(m, c, device="cuda", generator=g).to(dtype) for c in (k, n))
    w = torch.empty(1, 1, device="cuda", dtype=dtype).expand(n, k)
    dw = oztt.linear_backward(dy, x, w, need_input=False, need_bias=False)[1]
    for rows in torch.arange(n, device="cuda").split(512):
        want, mag = dy[:, rows].double().t() @ x.double(), dy[:, rows].double().abs().t() @ x.double().abs()
        tol = U[dtype] * want.abs() + 1.01 * m * 2.0 ** -23 * mag + TINY[dtype]
        assert bool(((dw[rows].double() - want).abs() <= tol).all())
