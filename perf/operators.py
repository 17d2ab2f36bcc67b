"""The measured calls of the training and serving operators: the matrix product with bias, activation and
residual in its epilogue (`linear`), its gradients (`linear_backward`) and the AdamW step over many tensors.

`run` computes each in its plain form (elementary torch operations in 32 bits, rounded once at the end), or,
where `own` is true, through the package's operators. `exact` is the definition in 64 bits.

The 8-bit states of AdamW: blocks of 256 elements share an exponent. A first moment is a sign and seven bits
(four of the exponent, three of the mantissa) below it, a second moment eight bits (five and three), rounded
stochastically with 16 random bits for each, hashed from the element's position and the step's seed. The plain
form keeps the same values in 32 bits; both sides return them in bfloat16, which holds every one exactly.
"""

import math

import torch

own = False

BLOCK = 256
HALF = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# 2 * 8192 * 4096 * 16384 * 2 multiplications and additions: the largest listed case
MOST_FLOPS = 4 * 8192 * 4096 * 16384
MOST_ELEMENTS = 16 * 4096 * 4096


def listed():
    return [
        # one token's output projection: serving at batch 1, where latency counts
        {"name": "token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "act": "none", "bias": True,
         "residual": True, "pre": False, "layout": "nk"},
        # a small batch of single tokens through the widening product of a feed-forward block
        {"name": "few tokens", "op": "linear", "m": 16, "n": 14080, "k": 3520, "dtype": "fp16", "act": "silu",
         "bias": False, "residual": False, "pre": False, "layout": "nk"},
        # a short prompt, every size odd, the weight stored transposed
        {"name": "odd prompt", "op": "linear", "m": 333, "n": 2047, "k": 1001, "dtype": "fp16", "act": "gelu",
         "bias": True, "residual": True, "pre": False, "layout": "kn"},
        # training forward through the widening product: keeps what its backward pass needs
        {"name": "widen", "op": "linear", "m": 2048, "n": 16384, "k": 4096, "dtype": "bf16", "act": "gelu_tanh",
         "bias": True, "residual": False, "pre": True, "layout": "nk"},
        # a long batch through the narrowing product back onto the residual stream
        {"name": "narrow", "op": "linear", "m": 8192, "n": 4096, "k": 16384, "dtype": "bf16", "act": "none",
         "bias": True, "residual": True, "pre": False, "layout": "nk"},
        # the backward pass of a small layer
        {"name": "small backward", "op": "backward", "m": 512, "n": 1024, "k": 1024, "dtype": "bf16", "act": "relu",
         "bias": True, "layout": "nk"},
        # a ragged batch, odd layer widths
        {"name": "odd backward", "op": "backward", "m": 777, "n": 1535, "k": 1001, "dtype": "fp16", "act": "silu",
         "bias": True, "layout": "nk"},
        # the backward pass of a long batch through the widening product
        {"name": "long backward", "op": "backward", "m": 8192, "n": 16384, "k": 4096, "dtype": "bf16",
         "act": "gelu_tanh", "bias": True, "layout": "nk"},
        # biases and gains only: many tensors of a few thousand elements, where launches would count
        {"name": "gains", "op": "adamw", "tensors": 24, "size": 2048, "param": "fp32", "grad": "fp32",
         "master": False, "bits": 32, "clip": False, "shift": 0},
        # a layer trained in bfloat16 with 32-bit master weights and states
        {"name": "layer", "op": "adamw", "tensors": 9, "size": 4096 * 1024, "param": "bf16", "grad": "bf16",
         "master": True, "bits": 32, "clip": True, "shift": 0},
        # hundreds of tensors of ragged sizes in a buffer that is not aligned, 8-bit states
        {"name": "ragged 8-bit", "op": "adamw", "tensors": 300, "size": 30011, "param": "bf16", "grad": "bf16",
         "master": False, "bits": 8, "clip": True, "shift": 1},
        # a whole stage's weights, 8-bit states
        {"name": "stage 8-bit", "op": "adamw", "tensors": 20, "size": 8192 * 1480, "param": "bf16", "grad": "bf16",
         "master": True, "bits": 8, "clip": False, "shift": 0},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "backward", "adamw"])
    if op == "adamw":
        while True:
            tensors, size = _spread(rng, 1, 400), _spread(rng, 64, 1 << 24)
            if tensors * size <= MOST_ELEMENTS // 2:
                break
        bits = rng.choice([8, 32])
        param = rng.choice(["bf16", "fp32", "fp16"])
        return {"op": op, "tensors": tensors, "size": size, "param": param,
                "grad": rng.choice(["fp32", param]), "master": param != "fp32" and rng.random() < 0.5, "bits": bits,
                "clip": rng.random() < 0.5, "shift": rng.choice([0, 0, 1])}
    while True:
        m, n, k = _spread(rng, 1, 16384), _spread(rng, 64, 16384), _spread(rng, 64, 16384)
        if rng.random() < 0.6:  # layer widths are mostly multiples of a power of two
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        if m * n * k * (2 if op == "linear" else 4) <= MOST_FLOPS:
            break
    case = {"op": op, "m": m, "n": n, "k": k, "dtype": rng.choice(["bf16", "fp16"]),
            "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.7,
            "layout": rng.choice(["nk", "nk", "nk", "kn"])}
    if op == "linear":
        case.update(residual=rng.random() < 0.5, pre=case["act"] != "none" and rng.random() < 0.5)
    return case


# ---- inputs ---------------------------------------------------------------------------------------------


def _sizes(case):
    """Ragged sizes around the typical one."""
    return [max(1, int(case["size"] * (0.25 + 1.5 * ((37 * i + 50) % 101) / 101.0))) for i in range(case["tensors"])]


def _offsets(sizes):
    at, total = [], 0
    for n in sizes:
        at.append(total)
        total += -(-n // BLOCK) * BLOCK
    return at, total


def _linear_inputs(case, g):
    m, n, k, dt = case["m"], case["n"], case["k"], HALF[case["dtype"]]
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    s = {"x": rand(m, k).to(dt)}
    if case["layout"] == "nk":
        s["w"] = (rand(n, k) / math.sqrt(k)).to(dt)
    else:  # stored with the output features side by side
        s["w"] = (rand(k, n) / math.sqrt(k)).to(dt).t()
    s["b"] = (0.1 * rand(n)).to(dt) if case["bias"] else None
    return s, rand, dt


def _adamw_inputs(case, g):
    sizes = _sizes(case)
    at, total = _offsets(sizes)
    shift = case["shift"]
    live = torch.zeros(total, dtype=torch.bool, device="cuda")  # false in the padding between tensors
    for n, o in zip(sizes, at):
        live[o:o + n] = True

    def flat(dtype, scale):
        buf = torch.zeros(total + shift, dtype=dtype, device="cuda")[shift:]
        v = torch.randn(total, device="cuda", generator=g) * scale
        # gradients of real layers differ in size from row to row: a factor for each block of elements
        return buf, torch.where(live, v, torch.zeros_like(v))

    s = {"sizes": sizes, "at": at, "t": 0}
    p, v = flat(HALF[case["param"]], 0.02)
    s["master"] = v.clone() if case["master"] else None
    s["p"] = p.copy_(v)
    gr, v = flat(HALF[case["grad"]], 1e-3)
    size = torch.exp(1.5 * torch.randn(total // BLOCK, device="cuda", generator=g))
    s["g"] = gr.copy_((v.view(-1, BLOCK) * size[:, None]).view(-1))
    s["scale"] = torch.full((1,), 0.73, device="cuda") if case["clip"] else None
    s["seed"] = int(torch.randint(0, 1 << 30, (1,), device="cuda", generator=g))
    s["hyper"] = {"lr": 3e-4, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1}
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "adamw":
        s = _adamw_inputs(case, g)
        total = s["p"].numel()
        pieces = lambda t: None if t is None else [t[o:o + n] for o, n in zip(s["at"], s["sizes"])]  # noqa: E731
        if own:  # the handle that a training program keeps: the parameters, their states and their layout
            import oztt_b200 as oz

            s["opt"] = oz.AdamW(pieces(s["p"]), masters=pieces(s["master"]), state_bits=case["bits"], **s["hyper"])
            s["grads"] = pieces(s["g"])
        else:
            s["m"], s["v"] = (torch.zeros(total, device="cuda") for _ in range(2))
    else:
        s, rand, dt = _linear_inputs(case, g)
        m, n = case["m"], case["n"]
        if case["op"] == "linear":
            s["r"] = rand(m, n).to(dt) if case["residual"] else None
        else:
            z = s["x"] @ s["w"].t()
            s["z"] = (z if s["b"] is None else z + s["b"]) if case["act"] != "none" else None
            s["dy"] = (0.05 * rand(m, n)).to(dt)
    s["case"] = case
    return s


# ---- the plain forms ------------------------------------------------------------------------------------


def _activate(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain_linear(s, case):
    dt = s["x"].dtype
    z = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _activate(z, case["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(dt), "pre": z.to(dt) if case["pre"] else None}


def _plain_backward(s, case):
    dt = s["x"].dtype
    dz = s["dy"].float()
    if case["act"] != "none":
        dz = dz * _slope(s["z"].float(), case["act"])
    return {"dx": (dz @ s["w"].float()).to(dt), "dw": (dz.t() @ s["x"].float()).to(dt),
            "db": dz.sum(0).to(dt) if case["bias"] else None}


def _random_bits(total, seed):
    """32 bits for each position: three multiplications and shifts, all modulo 2^32."""
    mask = 0xFFFFFFFF
    h = (torch.arange(total, device="cuda") * 0x9E3779B9 + seed) & mask
    h = ((h ^ (h >> 16)) * 0xBB67AE85) & mask
    h = ((h ^ (h >> 15)) * 0x6A09E667) & mask
    return h ^ (h >> 16)


def _to_8_bits(x, random, exponent_bits, floor):
    """The values that the 8-bit codes of x stand for."""
    top = (1 << exponent_bits) - 1
    bits = x.abs().view(torch.int32)
    base = ((bits.view(-1, BLOCK).amax(1, keepdim=True) + 0xFFFFF) >> 23) - top
    base = (torch.clamp(base, 0, 254 - top) << 3).expand(-1, BLOCK).reshape(-1)
    code = torch.clamp(((bits + random) >> 20) - base, 0, 8 * top + 7)
    if floor:  # what is not zero is not stored as zero
        code = torch.where(bits > 0, torch.clamp(code, min=1), code)
    return torch.copysign(torch.where(code > 0, (code + base) << 20, torch.zeros_like(code)).view(torch.float32), x)


def _plain_adamw(s, case):
    h = s["hyper"]
    (b1, b2), lr = h["betas"], h["lr"]
    s["t"] += 1
    g = s["g"].float()
    if s["scale"] is not None:
        g = g * s["scale"]
    m = b1 * s["m"] + (1 - b1) * g
    v = b2 * s["v"] + ((1 - b2) * g) * g
    p = (s["p"].float() if s["master"] is None else s["master"]) * (1 - lr * h["weight_decay"])
    p = p - (lr / (1 - b1 ** s["t"])) * (m / (torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** s["t"])) + h["eps"]))
    if s["master"] is not None:
        s["master"].copy_(p)
    s["p"].copy_(p)
    if case["bits"] == 8:
        r = _random_bits(m.numel(), s["seed"] + s["t"])
        m = _to_8_bits(m, ((r & 0xFFFF) << 4).to(torch.int32), 4, False)
        v = _to_8_bits(v, ((r >> 16) << 4).to(torch.int32), 5, True)
    s["m"], s["v"] = m, v
    kind = torch.bfloat16 if case["bits"] == 8 else torch.float32
    return {"p": s["p"], "master": s["master"], "m": m.to(kind), "v": v.to(kind)}


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"linear": _plain_linear, "backward": _plain_backward, "adamw": _plain_adamw}[case["op"]](s, case)
    import oztt_b200 as oz

    if case["op"] == "linear":
        out = oz.linear(s["x"], s["w"], s["b"], residual=s["r"], activation=case["act"], save_pre=case["pre"])
        return {"y": out[0], "pre": out[1]} if case["pre"] else {"y": out, "pre": None}
    if case["op"] == "backward":
        dx, dw, db = oz.linear_backward(s["dy"], s["x"], s["w"], pre=s["z"], activation=case["act"],
                                        need_bias=case["bias"])
        return {"dx": dx, "dw": dw, "db": db}
    s["t"] += 1
    s["opt"].step(s["grads"], grad_scale=s["scale"], seed=s["seed"] + s["t"])
    m, v = s["opt"].moments()
    return {"p": s["p"], "master": s["master"], "m": m, "v": v}


# ---- what is computed, and its definition in 64 bits ----------------------------------------------------


def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        p, g = (torch.empty(0, dtype=HALF[case[x]]).element_size() for x in ("param", "grad"))
        weights = 8 + p if case["master"] else 2 * p
        # states read and written; in 8 bits they are also returned in bfloat16
        states = 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4
        return {"bytes": n * (weights + g + states), "flops": 14 * n}
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "linear":
        return {"bytes": 2 * (m * k + n * k + m * n * (1 + case["residual"] + case["pre"]) + n * case["bias"]),
                "flops": 2 * m * n * k}
    return {"bytes": 2 * (2 * m * k + 2 * n * k + m * n * (1 + (case["act"] != "none")) + n * case["bias"]),
            "flops": 4 * m * n * k}


def _phi(z):
    """The normal distribution's cumulative function, without cancellation in its lower tail."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _exact_linear(s, case):
    z = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
    z = z if s["b"] is None else z.add_(s["b"].double())
    pre = z.clone() if case["pre"] else None
    act = case["act"]
    if act == "relu":
        z = torch.where(z > 0, z, 0.0)
    elif act == "gelu":
        z = z * _phi(z)
    elif act == "gelu_tanh":
        z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    elif act == "silu":
        z = z * torch.sigmoid(z)
    return {"y": z if s["r"] is None else z + s["r"].double(), "pre": pre}


def _exact_backward(s, case):
    act, dz = case["act"], s["dy"].double()
    if act != "none":
        z = s["z"].double()
        if act == "relu":
            slope = torch.where(z > 0, 1.0, 0.0).double()
        elif act == "gelu":
            slope = _phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        elif act == "gelu_tanh":
            c = 2 * math.sqrt(2 / math.pi)
            q = torch.sigmoid(c * (z + 0.044715 * z ** 3))
            slope = q + z * q * (1 - q) * c * (1 + 0.134145 * z ** 2)
        else:
            q = torch.sigmoid(z)
            slope = q + z * q * (1 - q)
        dz = dz * slope
    return {"dx": torch.einsum("mn,nk->mk", dz, s["w"].double()), "dw": torch.einsum("mn,mk->nk", dz, s["x"].double()),
            "db": torch.einsum("mn->n", dz) if case["bias"] else None}


def _exact_8_bits(x, random, exponent_bits, floor):
    """Rounds |x| to a multiple of an eighth of its binade, up with the random number's probability, within the
    range that the block's exponent leaves."""
    a = x.abs()
    ceil_binade = lambda y: torch.frexp(y)[1] - 1  # noqa: E731
    top = torch.clamp(ceil_binade(a.view(-1, BLOCK).amax(1, keepdim=True) * (1 + 0.125 * (1 - 2.0 ** -20))), min=-127)
    low = (top - ((1 << exponent_bits) - 1)).expand(-1, BLOCK).reshape(-1)
    step = torch.exp2((ceil_binade(torch.where(a > 0, a, 1.0)) - 3).double())
    q = torch.floor(a / step + random.double() / 2.0 ** 20) * step
    least = torch.exp2(low.double()) * 1.125
    q = torch.where(q < least * 0.99, torch.where((a > 0) & floor, least, 0.0), q)
    return torch.copysign(q, x)


def _exact_adamw(s, case):
    h = s["hyper"]
    (b1, b2), lr = h["betas"], h["lr"]
    g = s["g"].double()
    if s["scale"] is not None:
        g = g * s["scale"].double()
    m, v = (1 - b1) * g, (1 - b2) * g * g  # the states start at zero
    p = (s["p"] if s["master"] is None else s["master"]).double()
    p = p - lr * h["weight_decay"] * p - lr * (m / (1 - b1)) / (torch.sqrt(v / (1 - b2)) + h["eps"])
    if case["bits"] == 8:
        r = _random_bits(m.numel(), s["seed"] + 1)
        m, v = _exact_8_bits(m, (r & 0xFFFF) << 4, 4, False), _exact_8_bits(v, (r >> 16) << 4, 5, True)
    return {"p": p, "master": None if s["master"] is None else p, "m": m, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "backward": _exact_backward, "adamw": _exact_adamw}[case["op"]](s, case)
