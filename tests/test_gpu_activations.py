"""Activations at every finite value of the types, against their definitions in 64 bits.

With one term a sum is the weight itself. Tolerances, derived: 2^x and 1/x are within 2^-22 and every other operation
within 2^-24 of itself; the exponent of 2^x is at most 126 in size and has four roundings, so the exponential is within
126 * 4 * 2^-24 of itself, and the polynomial of the normal distribution within 2^-13.8: together, y is within 2^-13 of
itself, and once more rounded. A factor below 2^-126 is flushed to zero: beside |z| <= 13 (GELU, both forms) and
|z| <= 90 (SILU) that is 2^-122 and 2^-119 of y.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # the smallest subnormal
FLUSHED = {"relu": 0.0, "gelu": 2.0 ** -122, "gelu_tanh": 2.0 ** -122, "silu": 2.0 ** -119}
ACTS = ["relu", "gelu", "gelu_tanh", "silu"]


def finite(dtype):
    v = torch.arange(-2 ** 15, 2 ** 15, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    return v[torch.isfinite(v)]


def y64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
def test_every_value(oztt, cuda, dtype, act):
    z = finite(dtype)
    y, pre = oztt.linear(torch.ones(1, 1, device="cuda", dtype=dtype), z[:, None], activation=act, save_pre=True)
    assert torch.equal(pre[0], z)
    want = y64(z.double(), act)
    tol = U[dtype] * want.abs() + 2.0 ** -13 * (1 + U[dtype]) * want.abs() + FLUSHED[act] + TINY[dtype]
    off = ((y[0].double() - want).abs() / tol)
    assert bool((off <= 1).all()), f"worst {float(off.max()):.3g} of its tolerance at {float(z[off.argmax()])}"
