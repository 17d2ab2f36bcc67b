"""The layer operators under torch's tracers and dispatch modes: the right result, or an error."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu


def tensors(dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return r(40, 96), r(72, 96) / 8, r(72), r(40, 72)


def call(oztt, x, w, b, r):
    return oztt.linear(x, w, b, residual=r, activation="silu")


@pytest.mark.parametrize("grad", [False, True])
def test_traced(oztt, cuda, grad):
    t = tensors()
    other = [2 * x for x in t]
    t[1].requires_grad_(grad)
    f = torch.jit.trace(lambda *a: call(oztt, *a), t, check_trace=False)
    junk = [torch.full((40, 72), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(8)]
    del junk  # what fresh memory would hold
    assert torch.equal(f(*other), call(oztt, *other))


def test_traced_with_pre(oztt, cuda):
    t = tensors()[:3]
    other = [2 * x for x in t]
    f = torch.jit.trace(lambda *a: oztt.linear(*a, activation="gelu", save_pre=True), t, check_trace=False)
    junk = [torch.full((40, 72), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(8)]
    del junk
    assert all(torch.equal(a, b) for a, b in zip(f(*other), oztt.linear(*other, activation="gelu", save_pre=True)))


def test_traced_gradients(oztt, cuda):
    x, w, b, dy = tensors()
    def g(dy, x, w):
        return oztt.linear_backward(dy, x, w, pre=dy, activation="gelu_tanh")
    f = torch.jit.trace(g, (dy, x, w), check_trace=False)
    junk = [torch.full(s, 7.0, device="cuda", dtype=torch.bfloat16) for s in ((40, 96), (72, 96), (72,)) for _ in range(8)]
    del junk
    assert all(torch.equal(a, b) for a, b in zip(f(2 * dy, 2 * x, w), g(2 * dy, 2 * x, w)))


@pytest.mark.parametrize("mode", ["real", "fake"])
def test_recorded(oztt, cuda, mode):
    """A recorder of dispatched operations (and one over tensors without memory) sees the products."""
    t = tensors()
    other = [2 * x for x in t]
    f = make_fx(lambda *a: call(oztt, *a), tracing_mode=mode)(*t)
    junk = [torch.full((40, 72), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(8)]
    del junk
    assert torch.equal(f(*other), call(oztt, *other))


def test_recorded_training(oztt, cuda):
    """The recorded gradients of a product are those of the product."""
    t = tensors()
    other = [2 * x for x in t]

    def f(x, w, b, r):
        a = [v.detach().requires_grad_(True) for v in (x, w, b, r)]
        return torch.autograd.grad((call(oztt, *a) * r).sum(), a)

    g = make_fx(f)(*t)
    junk = [torch.full(s, 7.0, device="cuda", dtype=torch.bfloat16) for s in ((40, 72), (40, 96), (72, 96), (72,)) for _ in range(8)]
    del junk
    assert all(torch.equal(a, b) for a, b in zip(g(*other), f(*other)))


@pytest.mark.parametrize("grad", [False, True])
def test_under_a_mode_that_counts(oztt, cuda, grad):
    """What only looks on changes nothing."""
    from torch.utils.flop_counter import FlopCounterMode

    t = [x.requires_grad_(grad) for x in tensors()]
    want = call(oztt, *t)
    with FlopCounterMode(display=False):
        y = call(oztt, *t)
    assert torch.equal(y, want) and y.requires_grad == grad
    if grad:
        a = torch.autograd.grad(y, t, torch.ones_like(y))
        b = torch.autograd.grad(want, t, torch.ones_like(y))
        assert all(torch.equal(x, z) for x, z in zip(a, b))


def test_tensors_without_memory(oztt, cuda):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode() as mode:
        x, w = (mode.from_tensor(v) for v in tensors()[:2])
        y, pre = oztt.linear(x, w, activation="relu", save_pre=True)
        assert y.shape == pre.shape == (40, 72) and y.dtype == x.dtype and y.device == x.device
        dx, dw, db = oztt.linear_backward(y, x, w, need_bias=False)
        assert dx.shape == x.shape and dw.shape == w.shape and db is None


def test_transforms_of_func_are_refused(oztt, cuda):
    t = tensors()
    for transformed in (lambda: torch.func.grad(lambda x: call(oztt, x, *t[1:]).float().sum())(t[0]),
                        lambda: torch.func.jvp(lambda x: call(oztt, x, *t[1:]), (t[0],), (torch.ones_like(t[0]),)),
                        lambda: torch.func.vmap(lambda b: call(oztt, t[0], t[1], b, t[3]))(torch.stack([t[2]] * 3)),
                        lambda: torch.func.vmap(lambda x: oztt.linear_backward(t[3], x, t[1]))(torch.stack([t[0]] * 3))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            transformed()


def test_forward_mode_under_a_mode_is_refused(oztt, cuda):
    import torch.autograd.forward_ad as fwad
    from torch.utils.flop_counter import FlopCounterMode

    t = list(tensors())
    with fwad.dual_level(), FlopCounterMode(display=False), pytest.raises((RuntimeError, NotImplementedError)):
        t[0] = fwad.make_dual(t[0], torch.ones_like(t[0]))
        call(oztt, *t)
