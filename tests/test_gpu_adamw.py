"""AdamW over many tensors against its definition in 64 bits.

Tolerances of one step, derived: with e = 2^-24 the unit of a 32-bit rounding, m takes three roundings and v four,
beyond the coefficients' own (one each): |dm| <= 4 e (|b1 m| + |(1-b1) g|) and |dv| <= 6 e v'. The root and the
quotient are approximate to 2^-22 each; with half of dv's relative error, the sum with eps and the products, the
step is within 2^-20 of itself plus lr/(1-b1^t) |dm| / denominator, and p adds two roundings of itself. A parameter
of 16 bits is rounded once more, to half its spacing.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 0.0}
HYPER = dict(lr=3e-3, betas=(0.9, 0.97), eps=1e-8, weight_decay=0.1)


def tensors(sizes, dtype, seed=0, scale=1.0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for n in sizes:
        buf = torch.empty(n + offset, dtype=dtype, device="cuda")[offset:]
        out.append(buf.copy_(scale * torch.randn(n, device="cuda", generator=g)))
    return out


def piece(opt, flat, i):
    return flat[opt.offsets[i]:opt.offsets[i] + opt.params[i].numel()]


def step64(p, g, m, v, t, lr, betas, eps, weight_decay, scale=1.0):
    """The step, the new moments and the bounds on their 32-bit errors, in 64 bits."""
    b1, b2 = betas
    g = g * scale
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    dm = 4 * E * (b1 * m.abs() + (1 - b1) * g.abs()) + 2.0 ** -148
    dv = 6 * E * v2 + 2.0 ** -148
    c = lr / (1 - b1 ** t)
    denom = torch.sqrt(v2 / (1 - b2 ** t)) + eps
    move = c * m2 / denom
    p2 = p * (1 - lr * weight_decay) - move
    dp = 3 * E * p.abs() + 2.0 ** -20 * move.abs() + c * dm / denom + 2.0 ** -148
    return p2, m2, v2, dp, dm, dv


def within(got, want, tol, what):
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), f"{what}: worst {float((d / (tol + 1e-300)).max()):.3g} of its tolerance"


@pytest.mark.parametrize("param,grad,master", [(torch.float32, torch.float32, False), (torch.float32, torch.bfloat16, False),
                                               (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.bfloat16, True),
                                               (torch.float16, torch.float32, True), (torch.float16, torch.float16, False)])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_steps_of_32_bits(oztt, cuda, param, grad, master, offset):
    sizes = [1, 7, 8, 255, 256, 257, 5000, 8192, 8193, 70001]
    params = tensors(sizes, param, 1, 0.5, offset)
    masters = [p.float() for p in params] if master else None
    opt = oztt.AdamW(params, masters=masters, **HYPER)
    for t in (1, 2, 3):
        grads = tensors(sizes, grad, 10 + t, 0.01, offset)
        scale = torch.tensor([0.3], device="cuda") if t == 2 else None
        m0, v0 = (x.double().clone() for x in opt.moments())
        p0 = [(w if master else p).double().clone() for p, w in zip(params, masters or params)]
        opt.step(grads, grad_scale=scale)
        m1, v1 = opt.moments()
        for i in range(len(sizes)):
            p2, m2, v2, dp, dm, dv = step64(p0[i], grads[i].double(), piece(opt, m0, i), piece(opt, v0, i), t,
                                            scale=float(scale) if scale is not None else 1.0, **HYPER)
            within(piece(opt, m1, i), m2, dm, "m")
            within(piece(opt, v1, i), v2, dv, "v")
            if master:
                within(masters[i], p2, dp, "master")
                assert torch.equal(params[i], masters[i].to(param))
            else:
                within(params[i], p2, U[param] * p2.abs() + (1 + U[param]) * dp + TINY[param], "p")


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("offset", range(1, 9))
def test_every_alignment(oztt, cuda, bits, offset):
    """Parameters and gradients at every address give what aligned ones give, bit for bit, and nothing beside them is
    written."""
    sizes = [1, 255, 256, 300, 4096, 9001]
    runs = []
    for off in (0, offset):
        for dtype in (torch.bfloat16, torch.float32):
            params, grads = [], []
            for n, v, g in zip(sizes, tensors(sizes, dtype, 1), tensors(sizes, dtype, 2)):
                room = torch.full((n + 32,), 7.0, dtype=dtype, device="cuda")
                params.append(room[8 + off:8 + off + n].copy_(v))
                grads.append(torch.full((n + 32,), 7.0, dtype=dtype, device="cuda")[24 - off:24 - off + n].copy_(g))
            opt = oztt.AdamW(params, state_bits=bits, seed=3, **HYPER)
            for _ in range(2):
                opt.step(grads)
            for p, n in zip(params, sizes):
                whole = p._base
                beside = torch.cat([whole[:8 + off], whole[8 + off + n:]])
                assert bool((beside == 7.0).all())
            runs.append((params, *opt.moments()))
    for aligned, other in ((runs[0], runs[2]), (runs[1], runs[3])):
        assert all(torch.equal(a, b) for a, b in zip(aligned[0], other[0]))
        assert torch.equal(aligned[1], other[1]) and torch.equal(aligned[2], other[2])


def random_bits(n, seed):
    mask = np.uint64(0xFFFFFFFF)
    h = (np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B9) + np.uint64(seed & 0xFFFFFFFF)) & mask
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0xBB67AE85)) & mask
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(0x6A09E667)) & mask
    return (h ^ (h >> np.uint64(16))).astype(np.int64)


def encode(x, r, top, floor):
    """The values of the 8-bit codes of x (float32, whole blocks), by the definition of the format."""
    bits = np.abs(x).view(np.uint32).astype(np.int64).reshape(-1, 256)
    e = np.clip(((bits.max(1, keepdims=True) + 0xFFFFF) >> 23) - top, 0, 254 - top)
    c = np.clip(((bits + r.reshape(-1, 256) * 16) >> 20) - 8 * e, 0, 8 * top + 7)
    if floor:
        c = np.where(bits > 0, np.maximum(c, 1), c)
    return np.copysign(np.where(c > 0, (8 * e + c) << 20, 0).astype(np.uint32).view(np.float32).reshape(-1), x)


@pytest.mark.parametrize("param,master,offset", [(torch.float32, False, 0), (torch.bfloat16, True, 0), (torch.bfloat16, False, 3)])
def test_steps_of_8_bits(oztt, cuda, param, master, offset):
    """Every code of three steps is the definition's, bit for bit: the moments take the same 32-bit roundings in
    numpy. Gradients of very different sizes within a block reach the ends of the format's range."""
    sizes = [1, 300, 256, 9000, 40001]
    params = tensors(sizes, param, 1, 0.5, offset)
    opt = oztt.AdamW(params, masters=True if master else None, state_bits=8, **HYPER)
    total = opt.blocks * 256
    m = np.zeros(total, np.float32)
    v = np.zeros(total, np.float32)
    f = np.float32
    b1, b2 = HYPER["betas"]
    for t in (1, 2, 3):
        g = torch.Generator(device="cuda").manual_seed(t)
        grads = [(torch.randn(n, device="cuda", generator=g) * torch.exp(6 * torch.randn(n, device="cuda", generator=g))
                  * (torch.rand(n, device="cuda", generator=g) > 0.1)) for n in sizes]
        flat = np.zeros(total, np.float32)
        for i, gr in enumerate(grads):
            flat[opt.offsets[i]:opt.offsets[i] + sizes[i]] = gr.cpu().numpy()
        p0 = [(w if w is not None else p).double().clone() for p, w in zip(params, opt.masters)]
        m0, v0 = (x.double() for x in opt.moments())
        opt.step(grads, seed=77 + t)
        for i in range(len(sizes)):  # the step is taken with the moments before their rounding
            p2, _, _, dp, _, _ = step64(p0[i], grads[i].double(), piece(opt, m0, i), piece(opt, v0, i), t, **HYPER)
            if master:
                within(opt.masters[i], p2, dp, "master")
            else:
                within(params[i], p2, U[param] * p2.abs() + (1 + U[param]) * dp + TINY[param], "p")
        r = random_bits(total, 77 + t)
        m = encode(f(b1) * m + f(1 - b1) * flat, r & 0xFFFF, 15, False)
        v = encode(f(b2) * v + (f(1 - b2) * flat) * flat, r >> 16, 31, True)
        got_m, got_v = opt.moments()
        assert np.array_equal(got_m.float().cpu().numpy(), m)
        assert np.array_equal(got_v.float().cpu().numpy(), v)


def test_rounding_of_8_bits_is_unbiased(oztt, cuda):
    """The mean of the stored moments over many seeds is the moment: within 5 standard deviations, those of a
    rounding between two neighbours (at most 1/8 of the value apart: at most 1/16 of it), and the 2^-16 that the
    random numbers' 16 bits may lose of an eighth."""
    n, seeds = 512, 400
    g = tensors([n], torch.float32, 4)[0]
    opt = oztt.AdamW([torch.zeros(n, device="cuda")], state_bits=8, betas=(0.5, 0.75))
    sums = torch.zeros(2, n, dtype=torch.float64, device="cuda")
    for s in range(seeds):
        for b in (opt.m, opt.v, opt.m_exp, opt.v_exp):
            b.zero_()
        opt.step([g], seed=1000 + 7 * s)
        m, v = opt.moments()
        sums[0] += m.double()
        sums[1] += v.double()
    for mean, want in ((sums[0] / seeds, 0.5 * g.double()), (sums[1] / seeds, 0.25 * g.double() ** 2)):
        assert bool(((mean - want).abs() <= want.abs() * (5 / 16 / math.sqrt(seeds) + 2.0 ** -19)).all())


def test_moments_of_8_bits_decay(oztt, cuda):
    """With zero gradients the moments decay on average as in 32 bits, although a step of 0.1 % is far below the
    spacing of a code. After 500 steps of 0.999 the mean over 65536 elements is 0.6064 of the start; each element's
    random walk has steps of at most 1/16 of its value, so the mean is within 5 * sqrt(500) / 16 / 256 = 0.027."""
    n = 65536
    opt = oztt.AdamW([torch.zeros(n, device="cuda")], state_bits=8, betas=(0.999, 0.999), lr=0.0)
    opt.step([1 + torch.rand(n, device="cuda")])
    m0, v0 = (x.double() for x in opt.moments())
    for _ in range(500):
        opt.step([torch.zeros(n, device="cuda")])
    for x0, x1 in zip((m0, v0), opt.moments()):
        assert abs(float((x1.double() / x0).mean()) / 0.999 ** 500 - 1) <= 0.027


def test_8_bits_train(oztt, cuda):
    """A least-squares problem is solved as well as with 32-bit moments (to twice the loss)."""
    torch.manual_seed(0)
    a = torch.randn(512, 300, device="cuda")
    want = torch.randn(300, device="cuda")
    losses = []
    for bits in (32, 8):
        p = torch.zeros(300, device="cuda")
        opt = oztt.AdamW([p], lr=0.03, weight_decay=0.0, state_bits=bits)
        for _ in range(600):
            opt.step([a.t() @ (a @ (p - want)) / 512])
        losses.append(float(((a @ (p - want)) ** 2).mean()))
    assert losses[1] <= 2 * losses[0] + 1e-4, losses


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors(oztt, cuda, bits):
    """More tensors than one launch holds, empty ones and ones without a gradient among them, give what each tensor
    gives by itself (with 8 bits: on the same random numbers, those of its place in the flat moments)."""
    sizes = [(37 * i) % 700 for i in range(1400)]
    params, grads = tensors(sizes, torch.float32, 1), tensors(sizes, torch.float32, 2)
    grads = [None if i % 11 == 5 else g for i, g in enumerate(grads)]
    before = [p.clone() for p in params]
    opt = oztt.AdamW(params, state_bits=bits, seed=9, **HYPER)
    opt.step(grads)
    m, v = opt.moments()
    for i in list(range(0, 60)) + list(range(1170, 1260)):
        if grads[i] is None or not sizes[i]:
            assert torch.equal(params[i], before[i]) and not bool(piece(opt, m, i).any())
            continue
        p2, m2, v2, dp, dm, dv = step64(before[i].double(), grads[i].double(), torch.zeros(sizes[i], device="cuda").double(),
                                        torch.zeros(sizes[i], device="cuda").double(), 1, **HYPER)
        within(params[i], p2, dp, "p")
        within(piece(opt, m, i), m2, dm + (m2.abs() / 8 if bits == 8 else 0) + (2.0 ** -15 * m2.abs().max() if bits == 8 else 0), "m")
        within(piece(opt, v, i), v2, dv + (v2 / 8 if bits == 8 else 0) + (2.0 ** -30 * v2.max() if bits == 8 else 0), "v")


def test_repeatable_and_resumable(oztt, cuda):
    """The same seed gives the same run; a run resumed from its state goes on as it would have."""
    sizes = [1000, 70000]
    runs = []
    for _ in range(2):
        params = tensors(sizes, torch.bfloat16, 3)
        opt = oztt.AdamW(params, masters=True, state_bits=8, seed=5)
        for t in range(4):
            if t == 2:
                mid = {k: (v.clone() if torch.is_tensor(v) else [w.clone() for w in v] if isinstance(v, list) else v)
                       for k, v in opt.state_dict().items()}
                mid_params = [p.clone() for p in params]
            opt.step(tensors(sizes, torch.bfloat16, 20 + t))
        runs.append((params, opt))
    (a, oa), (b, ob) = runs
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(oa.m, ob.m) and torch.equal(oa.v, ob.v)
    c = oztt.AdamW(mid_params, masters=True, state_bits=8)
    c.load_state_dict(mid)
    for t in (2, 3):
        c.step(tensors(sizes, torch.bfloat16, 20 + t))
    assert all(torch.equal(x, y) for x, y in zip(a, mid_params)) and torch.equal(oa.m, c.m) and torch.equal(oa.v_exp, c.v_exp)


@pytest.mark.parametrize("bits", [8, 32])
def test_non_finite_gradient_stays_in_its_block(oztt, cuda, bits):
    n = 2048
    p = tensors([n], torch.float32, 1)[0]
    q = p.clone()
    g = tensors([n], torch.float32, 2)[0]
    h = g.clone()
    h[700], h[1500] = math.nan, math.inf
    a, b = oztt.AdamW([p], state_bits=bits, seed=1), oztt.AdamW([q], state_bits=bits, seed=1)
    a.step([g])
    b.step([h])
    assert bool(q[700].isnan()) and bool(q[1500].isnan())  # inf / sqrt(inf)
    rest = torch.ones(n, dtype=torch.bool)
    rest[700] = rest[1500] = False
    assert torch.equal(p[rest], q[rest])
    if bits == 8:
        rest[512:768] = rest[1280:1536] = False
    assert all(torch.equal(x[rest], y[rest]) for x, y in zip(a.moments(), b.moments()))


def test_zero_gradients_and_extremes(oztt, cuda):
    p = torch.ones(600, device="cuda")
    opt = oztt.AdamW([p], state_bits=8, lr=0.1, weight_decay=0.0)
    opt.step([torch.zeros(600, device="cuda")])
    assert torch.equal(p, torch.ones_like(p)) and not bool(opt.m.any()) and not bool(opt.v.any())
    g = torch.full((600,), 1e-20, device="cuda")
    g[::2] = 3e18
    opt.step([g])
    m, v = opt.moments()
    assert bool(torch.isfinite(p).all()) and bool(torch.isfinite(m).all()) and bool(torch.isfinite(v).all())
    assert bool((v[1:600:2] > 0).all() | (g[1] ** 2 * 0.001 == 0))


def test_step_uses_grad_attributes_and_other_streams(oztt, cuda):
    p = tensors([1000], torch.float32, 1)[0].requires_grad_(True)
    q = p.detach().clone()
    a, b = oztt.AdamW([p]), oztt.AdamW([q])
    version = p._version
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        (p * p).sum().backward()
        a.step()
    s.synchronize()
    b.step([2 * q])
    assert torch.equal(p.detach(), q) and p._version > version


def test_parameters_that_moved(oztt, cuda):
    """A parameter given other memory between steps is stepped where it lies now; one that changed its kind is
    refused, and nothing is stepped."""
    p = torch.ones(500, device="cuda")
    q = p.clone()
    g = tensors([500], torch.float32, 2)[0]
    a, b = oztt.AdamW([p]), oztt.AdamW([q])
    for opt in (a, b):
        opt.step([g])
    old = p.data
    kept = old.clone()
    p.data = p.data.clone()
    for opt in (a, b):
        opt.step([g])
    assert torch.equal(p, q) and torch.equal(old, kept)
    for other in (p.data.half(), p.data[:499], torch.zeros(1000, device="cuda")[::2]):
        before = p.data
        p.data = other
        with pytest.raises(ValueError):
            a.step([g])
        p.data = before
    assert a.t == 2 and torch.equal(p, q)


def test_refusals(oztt, cuda):
    p = torch.zeros(64, device="cuda")
    wide = torch.zeros(64, 2, device="cuda")
    for make in (lambda: oztt.AdamW([]), lambda: oztt.AdamW([p.cpu()]), lambda: oztt.AdamW([p.double()]),
                 lambda: oztt.AdamW([wide[:, 0]]), lambda: oztt.AdamW([p], state_bits=16),
                 lambda: oztt.AdamW([p, p]), lambda: oztt.AdamW([p[:40], p[39:]]),
                 lambda: oztt.AdamW([p], masters=[]), lambda: oztt.AdamW([p], masters=[p.half()]),
                 lambda: oztt.AdamW([p], masters=[p])):
        with pytest.raises(ValueError):
            make()
    opt = oztt.AdamW([p])
    one = torch.ones(1, device="cuda")
    for kw in (dict(grads=[]), dict(grads=[p[:63]]), dict(grads=[p.double()]), dict(grads=[p.cpu()]),
               dict(grads=[wide[:, 0]]), dict(grads=[p + 1], grad_scale=one.double()),
               dict(grads=[p + 1], grad_scale=one.cpu()), dict(grads=[p + 1], lr=math.nan),
               dict(grads=[p + 1], lr=-1.0)):
        with pytest.raises(ValueError):
            opt.step(**kw)
    assert opt.t == 0 and not bool(p.any())
    for kw in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=math.inf)):
        with pytest.raises(ValueError):
            oztt.AdamW([p], **kw).step([p + 1])
    with pytest.raises(ValueError):
        oztt.AdamW([p], state_bits=8).load_state_dict(opt.state_dict())
