"""BF16 values below 2^-126 keep their value through every kernel of the products: sums, biases, residuals, db."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def values(dtype):
    v = torch.arange(-2 ** 15, 2 ** 15, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v) & (v != 0)]
    return v[: v.numel() // 16 * 16]


# one row by 16-byte accesses and element by element, a few unaligned rows, few terms, tiles, pairs by rows
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 8), (1, 1024), (3, 5), (16, 1), (16, 64), (40, 72), (300, 8), (300, 64)])
def test_forward(oztt, cuda, dtype, m, k):
    z = values(dtype)
    w = torch.zeros(z.numel(), k, device="cuda", dtype=dtype)
    w[:, 0] = z
    x = torch.zeros(m, k, device="cuda", dtype=dtype)
    x[:, 0] = 1
    zero = torch.zeros_like(z)
    want = z.expand(m, -1)
    assert torch.equal(oztt.linear(x, w), want)
    assert torch.equal(oztt.linear(x, w, zero), want)
    assert torch.equal(oztt.linear(x, w, zero, residual=torch.zeros_like(want)), want)
    assert torch.equal(oztt.linear(torch.zeros_like(x), w, z), want)
    assert torch.equal(oztt.linear(torch.zeros_like(x), w, residual=want), want)
    y, pre = oztt.linear(x, w, activation="relu", save_pre=True)
    assert torch.equal(pre, want) and torch.equal(y, want.clamp(min=0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 2, 4, 8, 16, 300])
def test_backward(oztt, cuda, dtype, m):
    z = values(dtype)
    n = z.numel()
    x, dy = (torch.zeros(m, c, device="cuda", dtype=dtype) for c in (n, 256))
    x[m // 2], dy[m // 2] = z, 1
    w = torch.zeros(256, n, device="cuda", dtype=dtype)
    w[0] = z
    dx, dw, _ = oztt.linear_backward(dy, x, w, need_bias=False)
    assert torch.equal(dw, z.expand(256, n)) and torch.equal(dx, dy[:, :1] * z)
    dy = torch.zeros(m, n, device="cuda", dtype=dtype)
    dy[m // 2] = z
    pre = torch.full_like(dy, 0.5)
    for act in ("none", "relu"):
        _, dw, db = oztt.linear_backward(dy, dy[:, :8] * 0 + 1, w.t()[:, :8], pre=pre, activation=act, need_input=False)
        assert torch.equal(db, z) and torch.equal(dw, z[:, None].expand(n, 8))
