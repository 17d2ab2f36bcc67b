"""Infinities and NaN through each kernel of the products reach their own row and column only."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# one token, a few unaligned rows, few rows, tiles, tiles of a shared sum, pairs by rows and with a residual
FORWARD = [(1, 264, 1024, False), (3, 129, 77, False), (16, 256, 4096, False), (40, 200, 128, True), (200, 264, 2048, False),
           (1300, 2064, 264, False), (1300, 2064, 264, True), (1301, 2065, 333, False)]


def make(m, n, k, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return r(m, k), r(n, k) / 8, r(n), r(m, n)


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0, 1e30, -1e30), b.nan_to_num(0.0, 1e30, -1e30))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,res", FORWARD)
def test_forward(oztt, cuda, m, n, k, res, dtype):
    x, w, b, r = make(m, n, k, dtype)
    r = r if res else None
    clean = oztt.linear(x, w, b, residual=r)
    bad = [(m - 1, k - 1, math.nan), (m // 2, 0, math.inf)][:1 if m == 1 else 2]
    x2, w2 = x.clone(), w.clone()
    for i, t, v in bad:
        x2[i, t] = v
    y = oztt.linear(x2, w, b, residual=r)
    rows = torch.ones(m, dtype=torch.bool, device="cuda")
    rows[[i for i, _, _ in bad]] = False
    assert torch.equal(y[rows], clean[rows]) and bool(y[m - 1].isnan().all())
    if m > 1:
        assert torch.equal(y[m // 2] == math.inf, w[:, 0] > 0) and torch.equal(y[m // 2] == -math.inf, w[:, 0] < 0)
    w2[n - 1, k // 2], w2[0, 0] = math.nan, -math.inf
    y = oztt.linear(x, w2, b, residual=r)
    assert torch.equal(y[:, 1:-1], clean[:, 1:-1]) and bool(y[:, -1].isnan().all())
    assert torch.equal(y[:, 0] == math.inf, x[:, 0] < 0) and torch.equal(y[:, 0] == -math.inf, x[:, 0] > 0)


# dw of few terms, of tiles and of pairs; dz by 16-byte accesses and element by element
BACKWARD = [(1, 264, 520), (4, 264, 520), (8, 1032, 264), (70, 96, 80), (333, 255, 129), (1500, 2000, 1704)]


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,n,k", BACKWARD)
def test_backward(oztt, cuda, m, n, k, act):
    x, w, b, dy = make(m, n, k)
    pre = dy.roll(1, 1)
    clean = oztt.linear_backward(dy, x, w, pre=pre, activation=act)
    i, j = m - 1, n // 2
    pre[i, j] = 1.0  # a slope that is not zero
    clean = oztt.linear_backward(dy, x, w, pre=pre, activation=act)
    bad = dy.clone()
    bad[i, j] = math.nan
    dx, dw, db = oztt.linear_backward(bad, x, w, pre=pre, activation=act)
    assert bool(dx[i].isnan().all()) and torch.equal(dx[:i], clean[0][:i])
    other = torch.arange(n, device="cuda") != j
    assert bool(dw[j].isnan().all()) and torch.equal(dw[other], clean[1][other])
    assert bool(db[j].isnan()) and torch.equal(db[other], clean[2][other])
    bad[i, j] = math.inf
    db = oztt.linear_backward(bad, x, w, pre=pre, activation=act)[2]
    assert float(db[j]) == math.inf and torch.equal(db[other], clean[2][other])
    x2 = x.clone()
    x2[i, 0] = math.nan
    _, dw, _ = oztt.linear_backward(dy, x2, w, pre=pre, activation=act)
    assert bool(dw[:, 0].isnan().all()) and torch.equal(dw[:, 1:], clean[1][:, 1:])
