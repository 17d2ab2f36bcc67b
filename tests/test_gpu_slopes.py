"""The activations' slopes at every finite value of the types, against their definitions in 64 bits.

With one row and one term, db and dw are dy times the slope. Tolerance, derived: 2^x and 1/x are within 2^-22 and every
other operation within 2^-24 of itself, and the slope is a sum of terms of at most 1.2 in size, where the exponent of 2^x
is below 10: within 2^-18, and exactly 0 or 1 from |z| = 128 on.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # the smallest subnormal
ACTS = ["relu", "gelu", "gelu_tanh", "silu"]


def finite(dtype):
    v = torch.arange(-2 ** 15, 2 ** 15, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    return v[torch.isfinite(v)]


def slope64(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi) if act == "gelu_tanh" else 1.0
    q = 0.044715 if act == "gelu_tanh" else 0.0
    s = torch.sigmoid(c * (z + q * z ** 3))
    return s + (s * (1 - s)) * (z * c * (1 + 3 * q * z * z))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
def test_every_slope(oztt, cuda, dtype, act):
    z = finite(dtype)
    one = torch.ones(1, 1, device="cuda", dtype=dtype)
    _, dw, db = oztt.linear_backward(torch.ones_like(z)[None], one, z[:, None], pre=z[None], activation=act, need_input=False)
    want = slope64(z.double(), act)
    for got in (db, dw[:, 0]):
        off = (got.double() - want).abs() - (U[dtype] * want.abs() + 2.0 ** -18 + TINY[dtype])
        assert bool((off <= 0).all()), f"{float(off.nan_to_num(math.inf).max()):.3g} beyond, at {float(z[off.nan_to_num(math.inf).argmax()])}"
        far = z.abs() >= 128
        assert torch.equal(got[far], (z[far] > 0).to(dtype))


@pytest.mark.parametrize("act", ACTS)
def test_slope_of_nan(oztt, cuda, act):
    """A sum that is NaN has no slope (RELU's, a comparison, is 0)."""
    z = torch.full((1, 64), math.nan, device="cuda", dtype=torch.bfloat16)
    one = torch.ones(1, 1, device="cuda", dtype=torch.bfloat16)
    db = oztt.linear_backward(torch.ones_like(z), one, z.t(), pre=z, activation=act, need_input=False, need_weight=False)[2]
    assert bool((db == 0).all() if act == "relu" else db.isnan().all())
