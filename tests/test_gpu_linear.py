"""The product of a layer with its epilogue, and its gradients, against their definitions in 64 bits.

Tolerances are derived: u is half the spacing of the output's type relative to its value (2^-8 for BF16, 2^-11 for
FP16), plus the smallest subnormal. Every output is rounded once (u |value|); the
32-bit sum of k products, of which the tensor core may drop low bits when it aligns its addends, is within
k 2^-23 of the sum S of the products' magnitudes; activations in 32 bits add 2^-20 |z| and scale the sum's error by
at most 1.13 (the largest slope of the GELU family). In the backward pass dz is rounded once more: u S for the
products.
"""

import math
import struct

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    z = z.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        g, = torch.autograd.grad(act64(z, act).sum(), z)
    return g


def make(m, n, k, dtype, seed=0, layout="plain"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, w = r(m, k).to(dtype), (r(n, k) / math.sqrt(max(k, 1))).to(dtype)
    if layout == "transposed":
        x, w = x.t().contiguous().t(), w.t().contiguous().t()
    elif layout == "padded":  # rows of a wider buffer, starting inside it
        bx, bw = r(m, k + 24).to(dtype), r(n, k + 16).to(dtype)
        bx[:, 8:8 + k], bw[:, 8:8 + k] = x, w
        x, w = bx[:, 8:8 + k], bw[:, 8:8 + k]
    elif layout == "odd offset":
        bx, bw = r(m * k + 1).to(dtype), r(n * k + 3).to(dtype)
        bx[1:], bw[3:] = x.reshape(-1), w.reshape(-1)
        x, w = bx[1:].view(m, k), bw[3:].view(n, k)
    elif layout == "every second":
        bx, bw = r(m, 2 * k).to(dtype), r(n, 2 * k).to(dtype)
        bx[:, ::2], bw[:, ::2] = x, w
        x, w = bx[:, ::2], bw[:, ::2]
    return x, w, (0.5 * r(n)).to(dtype), r(m, n).to(dtype)


def within(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = d > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol).max()):.3g} of its tolerance"


def check_forward(oztt, x, w, b, r, act, pre=False):
    dt = x.dtype
    out = oztt.linear(x, w, b, residual=r, activation=act, save_pre=pre)
    y, z = out if pre else (out, None)
    assert y.shape == x.shape[:-1] + (w.shape[0],) and y.dtype == dt and y.is_contiguous()
    k = w.shape[1]
    z64 = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z64, mag = z64 + b.double(), mag + b.double().abs()
    err = (k + 2) * 2.0 ** -23 * mag
    y64 = act64(z64, act)
    if pre:
        within(z, z64, U[dt] * z64.abs() + (1 + U[dt]) * err + TINY[dt], "pre")
    terr = 1.13 * err + 2.0 ** -20 * z64.abs()
    if r is not None:
        y64 = y64 + r.double()
        terr = terr + 2.0 ** -23 * y64.abs()
    within(y, y64, U[dt] * y64.abs() + (1 + U[dt]) * terr + TINY[dt], "y")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 64), (1, 4096, 1024), (2, 130, 72), (16, 256, 2048),
                                   (17, 255, 129), (32, 64, 4096), (33, 512, 520), (64, 1000, 256), (65, 129, 65),
                                   (128, 128, 128), (129, 384, 1000), (300, 777, 333), (512, 1024, 4096)])
def test_forward_sizes(oztt, cuda, dtype, m, n, k):
    x, w, b, r = make(m, n, k, dtype, seed=m + n + k)
    check_forward(oztt, x, w, b, r, "gelu", pre=True)
    check_forward(oztt, x, w, None, None, "none")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1500, 2000, 64), (2048, 2304, 200), (1281, 3001, 333), (2600, 1800, 1000),
                                   (20000, 264, 136), (300, 9000, 72)])
def test_forward_large(oztt, cuda, dtype, m, n, k):
    """Outputs of many tiles, whole and ragged, with every part of the epilogue."""
    x, w, b, r = make(m, n, k, dtype, seed=m + n + k)
    check_forward(oztt, x, w, b, r, "gelu_tanh", pre=True)
    check_forward(oztt, x, w, b, r[:, :1].expand(m, n), "relu")
    check_forward(oztt, x, w, None, None, "none")


@pytest.mark.parametrize("layout", ["transposed", "padded", "odd offset"])
def test_forward_large_layouts(oztt, cuda, layout):
    x, w, b, r = make(1700, 2100, 264, torch.bfloat16, seed=2, layout=layout)
    check_forward(oztt, x, w, b, r.t().contiguous().t(), "silu", pre=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k", [(300, 77), (1, 4097), (5, 16390), (2049, 515)])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
def test_forward_few_rows_unaligned(oztt, cuda, dtype, m, n, k):
    x, w, b, r = make(m, n, k, dtype, seed=m)
    check_forward(oztt, x, w, b, r, "silu", pre=True)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 9])
def test_backward_few_rows(oztt, cuda, m):
    x, w, b, dy = make(m, 520, 264, torch.bfloat16, seed=m)
    check_backward(oztt, dy, x, w, dy.roll(1, 1), "gelu")
    x, w, b, dy = make(m, 515, 77, torch.float16, seed=m)
    check_backward(oztt, dy, x, w, None, "none")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 6, 7, 8])
def test_sums_of_few_terms(oztt, cuda, dtype, m):
    for n, k in ((264, 520), (1, 8), (129, 1048)):
        x, w, b, dy = make(m, n, k, dtype, seed=m)
        check_backward(oztt, dy, x, w, None, "none")
    x, w, b, r = make(203, 264, m, dtype, seed=m)
    check_forward(oztt, x, w.t().contiguous().t(), None, None, "none")


@pytest.mark.parametrize("blocks", [3, 4, 6, 7, 9, 10, 12, 14, 31, 33])
@pytest.mark.parametrize("m", [5, 30, 64, 200])
def test_sums_shared_by_any_number(oztt, cuda, m, blocks):
    """Sums of `blocks` stretches of 64 terms (the last one short), shared by 1 to 8 or by 16 blocks of the device."""
    x, w, b, r = make(m, 200, 64 * blocks - 24, torch.bfloat16, seed=blocks)
    check_forward(oztt, x, w, b, r, "relu", pre=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1700, 2096, 40), (2049, 1536, 264), (1531, 2064, 1096)])
def test_forward_large_without_residual(oztt, cuda, dtype, act, m, n, k):
    x, w, b, r = make(m, n, k, dtype, seed=k)
    check_forward(oztt, x, w, b, None, act, pre=act != "relu")
    check_forward(oztt, x, w.t().contiguous().t(), None, None, act)


@pytest.mark.parametrize("n", [2064, 2065, 2079, 2090])
@pytest.mark.parametrize("offset", [0, 8, 16])
def test_outputs_inside_wider_ones(oztt, cuda, n, offset):
    """y and pre as columns of wider matrices, through the C ABI: their values, and nothing beside them written."""
    m, k, ld, dt = 1700, 136, 2112, torch.bfloat16
    x, w, b, _ = make(m, n, k, dt, seed=n)
    bufs = [torch.full((m, ld), 7.0, dtype=dt, device="cuda") for _ in range(2)]
    y, pre = (t[:, offset:offset + n] for t in bufs)
    views = [(t.data_ptr(), t.stride(0), t.stride(1)) for t in (x, w)] + [(b.data_ptr(), 0, 1), (0, 0, 0)]
    views += [(t.data_ptr(), ld, 1) for t in (y, pre)]
    args = struct.pack("=ii3Q" + 6 * "Qqq", 0, 0, m, n, k, *(v for view in views for v in view))
    oztt.call("oztt_linear_forward", 0, args, torch.cuda.current_stream().cuda_stream)
    want = x.double() @ w.double().t() + b.double()
    err = (k + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    for t, whole in ((y, bufs[0]), (pre, bufs[1])):
        within(t, want, U[dt] * want.abs() + (1 + U[dt]) * err + TINY[dt], "y and pre")
        assert bool((whole[:, :offset] == 7).all()) and bool((whole[:, offset + n:] == 7).all())


@pytest.mark.parametrize("n", [1, 2, 7, 8, 16, 17, 24, 32, 33])
@pytest.mark.parametrize("m", [1, 2, 9, 70, 300])
def test_backward_narrow(oztt, cuda, m, n):
    """Few output features: dz is a scratch matrix with as few columns, read across its rows for dw."""
    for k in (8, 1, 200):
        x, w, b, dy = make(m, n, k, torch.bfloat16, seed=m + n)
        check_backward(oztt, dy, x, w, dy.roll(1, 0), "silu")
        check_backward(oztt, dy, x, w, None, "none")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_forward_activations(oztt, cuda, act, dtype):
    x, w, b, r = make(96, 264, 192, dtype)
    for bias in (None, b):
        for res in (None, r):
            check_forward(oztt, 3 * x, w, bias, res, act, pre=True)


@pytest.mark.parametrize("layout", ["transposed", "padded", "odd offset", "every second"])
@pytest.mark.parametrize("m,n,k", [(1, 320, 256), (5, 77, 91), (200, 264, 136), (131, 255, 77)])
def test_forward_layouts(oztt, cuda, layout, m, n, k):
    x, w, b, r = make(m, n, k, torch.bfloat16, seed=5, layout=layout)
    check_forward(oztt, x, w, b, r.t().contiguous().t(), "silu", pre=True)
    check_forward(oztt, x, w, b[:1].expand(n), r[:1].expand(m, n), "none")


def test_forward_batch_dimensions(oztt, cuda):
    x, w, b, r = make(6 * 5, 96, 80, torch.float16)
    check_forward(oztt, x.view(6, 5, 80), w, b, r.view(6, 5, 96), "relu")
    check_forward(oztt, x.view(6, 5, 80).transpose(0, 1), w, b, r.view(6, 5, 96).transpose(0, 1), "relu")
    y = oztt.linear(x[0], w, b)
    assert y.shape == (96,) and torch.equal(y, oztt.linear(x[:1], w, b)[0])


def test_forward_empty(oztt, cuda):
    x, w, b, r = make(4, 96, 80, torch.bfloat16)
    assert oztt.linear(x[:0], w, b).shape == (0, 96)
    assert oztt.linear(x, w[:0], b[:0]).shape == (4, 0)
    y = oztt.linear(x[:, :0], w[:, :0], b, residual=r, activation="relu")  # an empty sum: the bias alone
    assert torch.equal(y, (b.float().clamp(min=0) + r.float()).to(y.dtype))


@pytest.mark.parametrize("act", ACTS)
def test_forward_infinities_and_nan(oztt, cuda, act):
    """An infinity or NaN reaches its own row and column only."""
    x, w, b, _ = make(40, 200, 128, torch.bfloat16)
    clean = oztt.linear(x, w, b, activation=act)
    x2 = x.clone()
    x2[3, 5], x2[17, 0] = math.inf, math.nan
    y = oztt.linear(x2, w, b, activation=act)
    rows = torch.tensor([i not in (3, 17) for i in range(40)])
    assert torch.equal(y[rows], clean[rows])
    assert bool(y[17].isnan().all())
    z = x2[3].double() @ w.double().t()
    assert bool((y[3][z > 0] == math.inf).all())
    if act == "none":
        assert bool((y[3][z < 0] == -math.inf).all())
    if act == "relu":
        assert bool((y[3][z < 0] == 0).all())


def test_forward_is_repeatable(oztt, cuda):
    for m, n, k in [(1, 512, 4096), (64, 256, 8192), (700, 900, 600)]:
        x, w, b, r = make(m, n, k, torch.bfloat16)
        y = oztt.linear(x, w, b, residual=r, activation="gelu")
        for _ in range(5):
            assert torch.equal(y, oztt.linear(x, w, b, residual=r, activation="gelu"))


def test_forward_on_another_stream(oztt, cuda):
    x, w, b, r = make(128, 512, 1024, torch.bfloat16)
    want = oztt.linear(x, w, b, residual=r)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x2 = x * 1  # ordered on s, ahead of the product
        y = oztt.linear(x2, w, b, residual=r)
    s.synchronize()
    assert torch.equal(y, want)


def test_forward_in_a_graph(oztt, cuda):
    x, w, b, r = make(8, 512, 520, torch.bfloat16)
    xo, wo, _, _ = make(8, 512, 519, torch.bfloat16)  # needs a packed copy
    oztt.linear(x, w, b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = oztt.linear(x, w, b, residual=r)
        yo = oztt.linear(xo, wo, b)
    x.mul_(2)
    xo.mul_(2)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, oztt.linear(x, w, b, residual=r)) and torch.equal(yo, oztt.linear(xo, wo, b))


def check_backward(oztt, dy, x, w, z, act, **need):
    dt = x.dtype
    dx, dw, db = oztt.linear_backward(dy, x, w, pre=z, activation=act, **need)
    m, (n, k) = x.shape[0], w.shape
    dz = dy.double()
    derr = torch.zeros_like(dz)  # of dz in 32 bits
    if act != "none":
        s = slope64(z.double(), act)
        # the slope in 32 bits: its terms are at most 1 + |z| in size
        derr = dz.abs() * 2.0 ** -20 * (1 + z.double().abs())
        dz = dz * s
    rounded = (U[dt] * dz.abs() + TINY[dt] if act != "none" else 0 * dz) + derr
    if dx is not None:
        want, mag, re = dz @ w.double(), dz.abs() @ w.double().abs(), rounded @ w.double().abs()
        within(dx, want, U[dt] * want.abs() + 1.01 * (re + (n + 2) * 2.0 ** -23 * mag) + TINY[dt], "dx")
    if dw is not None:
        want, mag, re = dz.t() @ x.double(), dz.t().abs() @ x.double().abs(), rounded.t() @ x.double().abs()
        within(dw, want, U[dt] * want.abs() + 1.01 * (re + (m + 2) * 2.0 ** -23 * mag) + TINY[dt], "dw")
    if db is not None:
        want = dz.sum(0)
        within(db, want, U[dt] * want.abs() + 1.01 * (derr.sum(0) + (m + 2) * 2.0 ** -24 * dz.abs().sum(0)) + TINY[dt], "db")
    return dx, dw, db


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 256, 128), (7, 130, 66), (64, 192, 320), (130, 255, 129),
                                   (333, 512, 264), (1024, 384, 640)])
def test_backward_sizes(oztt, cuda, act, dtype, m, n, k):
    x, w, b, dy = make(m, n, k, dtype, seed=m)
    z = (2 * dy.float().roll(1, 0) * dy.float().roll(1, 1)).to(dtype)
    check_backward(oztt, dy, x, w, z if act != "none" else None, act)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1500, 2000, 1700), (2048, 256, 2304), (1281, 3001, 1333), (5000, 520, 2600)])
def test_backward_large(oztt, cuda, dtype, m, n, k):
    x, w, b, dy = make(m, n, k, dtype, seed=m)
    z = (2 * dy.float().roll(1, 0) * dy.float().roll(1, 1)).to(dtype)
    check_backward(oztt, dy, x, w, z, "gelu_tanh")
    check_backward(oztt, dy, x, w, None, "none")


@pytest.mark.parametrize("layout", ["transposed", "padded", "odd offset", "every second"])
@pytest.mark.parametrize("m,n,k", [(5, 77, 91), (200, 264, 136)])
def test_backward_layouts(oztt, cuda, layout, m, n, k):
    x, w, b, dy = make(m, n, k, torch.bfloat16, seed=9, layout=layout)
    z = dy.roll(1, 0).t().contiguous().t()
    check_backward(oztt, dy, x, w, z, "gelu")
    check_backward(oztt, dy.t().contiguous().t(), x, w, None, "none")
    check_backward(oztt, dy[:1].expand(m, n), x, w, None, "none")


def test_backward_parts(oztt, cuda):
    x, w, b, dy = make(70, 96, 80, torch.bfloat16)
    z = dy.roll(1, 0)
    whole = oztt.linear_backward(dy, x, w, pre=z, activation="silu")
    for i in range(3):
        need = dict(need_input=i == 0, need_weight=i == 1, need_bias=i == 2)
        part = oztt.linear_backward(dy, x, w, pre=z, activation="silu", **need)
        assert all((p is None) == (j != i) for j, p in enumerate(part)) and torch.equal(part[i], whole[i])


def test_backward_empty(oztt, cuda):
    x, w, b, dy = make(4, 96, 80, torch.bfloat16)
    dx, dw, db = oztt.linear_backward(dy[:0], x[:0], w)
    assert dx.shape == (0, 80) and not bool(dw.any()) and not bool(db.any())
    dx, dw, db = oztt.linear_backward(dy[:, :0], x, w[:0])
    assert not bool(dx.any()) and dw.shape == (0, 80) and db.shape == (0,)
    dx, dw, db = oztt.linear_backward(dy, x[:, :0], w[:, :0])
    assert dx.shape == (4, 0) and dw.shape == (96, 0)
    check_backward(oztt, dy, x, w, None, "none")


@pytest.mark.parametrize("act", ACTS)
def test_autograd(oztt, cuda, act):
    """Through torch's autograd: the same gradients as linear_backward's, the residual's is dy."""
    x, w, b, r = make(48, 72, 64, torch.float16)
    dy = torch.randn_like(r)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = oztt.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act)
    y.backward(dy)
    z = oztt.linear(x, w, b)
    want = oztt.linear_backward(dy, x, w, pre=z if act != "none" else None, activation=act)
    for leaf, g in zip(leaves, (*want, dy)):
        assert torch.equal(leaf.grad, g)


@pytest.mark.parametrize("act", ACTS)
def test_gradient_against_differences(oztt, cuda, act):
    """Along a random direction v of each input, the change of L = sum(y dy) over a step. The step h is large enough
    for the type's rounding: y is rounded to u |y|, so the difference quotient is off by the rounding of two sums
    of mn outputs, at most 2 u sum |y dy| / (2h) but random in sign: taken as 4 standard deviations,
    4 u sqrt(sum (y dy)^2) / h. The third derivative's share is h^2 sum |dy| max|z'|^3 (below 2 |z'|^3 for
    these activations; RELU, which has a kink, is compared on inputs away from it)."""
    dt = torch.float16
    m, n, k = 24, 40, 32
    x, w, b, _ = make(m, n, k, dt, seed=3)
    if act == "relu":  # no sum near zero: the bias decides
        b = torch.where(b > 0, 20.0, -20.0).to(dt)
    dy = torch.randn(m, n, device="cuda").to(dt)
    z = oztt.linear(x, w, b)
    dx, dw, db = oztt.linear_backward(dy, x, w, pre=z if act != "none" else None, activation=act)
    h = 2.0 ** -4
    for name, g in (("x", dx), ("w", dw), ("b", db)):
        t = {"x": x, "w": w, "b": b}[name]
        v = torch.randint(0, 2, t.shape, device="cuda").to(dt) * 2 - 1
        val = []
        for sgn in (1, -1):
            a = {"x": x, "w": w, "b": b}
            a[name] = (t.double() + sgn * h * v.double()).to(dt)
            y = oztt.linear(a["x"], a["w"], a["b"], activation=act)
            val.append((y.double() * dy.double()).sum())
        a = {"x": x.double(), "w": w.double(), "b": b.double()}
        step = ((t.double() + h * v.double()).to(dt).double() - (t.double() - h * v.double()).to(dt).double()) / 2
        zdot = {"x": lambda: step @ a["w"].t(), "w": lambda: a["x"] @ step.t(), "b": lambda: step.expand(m, n)}[name]()
        want = float((g.double() * step).sum())
        spread = U[dt] * float(((act64(z.double(), act) * dy.double()) ** 2).sum()) ** 0.5
        rounding = U[dt] * float((g.double() * step).abs().sum())
        curve = 2 * float((dy.double().abs() * zdot.abs() ** 3).sum())
        assert abs(float(val[0] - val[1]) / 2 - want) <= 4 * spread + rounding + curve, name


def test_a_wait_that_gave_up_is_reported_once(oztt, cuda):
    x, w, b, r = make(8, 96, 80, torch.bfloat16)
    want = oztt.linear(x, w, b)
    oztt.call("oztt_test_linear_error", 2)
    with pytest.raises(RuntimeError, match="earlier call gave up waiting"):
        oztt.linear(x, w, b)
    assert torch.equal(oztt.linear(x, w, b), want)


def test_refusals(oztt, cuda):
    x, w, b, r = make(4, 96, 80, torch.bfloat16)
    bad = [lambda: oztt.linear(x.float(), w.float()), lambda: oztt.linear(x, w.half()), lambda: oztt.linear(x.cpu(), w),
           lambda: oztt.linear(x, w[:, :79]), lambda: oztt.linear(x, w, b[:95]), lambda: oztt.linear(x, w, b.float()),
           lambda: oztt.linear(x, w, residual=r[:3]), lambda: oztt.linear(x, w, activation="tanh"),
           lambda: oztt.linear(x, w, residual=r[:1]), lambda: oztt.linear(x, w.view(2, 48, 80)),
           lambda: oztt.linear_backward(r, x, w, activation="gelu"), lambda: oztt.linear_backward(r[:3], x, w),
           lambda: oztt.linear_backward(r, x, w, pre=r[:, :95], activation="gelu"),
           lambda: oztt.linear_backward(r.half(), x, w), lambda: oztt.linear_backward(r, x, w, activation="sigmoid")]
    for call in bad:
        with pytest.raises(ValueError):
            call()
