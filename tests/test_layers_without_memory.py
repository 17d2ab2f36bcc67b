"""The layer products on tensors that have a shape and no memory (on any machine): what they give, and that a recorder
finds them."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device="cuda")


def test_linear(oztt, fake):
    x, w = fake(5, 8, 96), fake(72, 96)
    y, pre = oztt.linear(x, w, activation="relu", save_pre=True)
    assert y.shape == pre.shape == (5, 8, 72) and y.dtype == x.dtype and y.device == x.device
    assert oztt.linear(x, w, fake(72), residual=y).shape == y.shape


def test_linear_backward(oztt, fake):
    x, w, dy = fake(40, 96), fake(72, 96), fake(40, 72)
    dx, dw, db = oztt.linear_backward(dy, x, w, pre=dy, activation="silu")
    assert (dx.shape, dw.shape, db.shape) == ((40, 96), (72, 96), (72,))
    dx, dw, db = oztt.linear_backward(dy, x, w, need_input=False, need_bias=False)
    assert dx is None and dw.shape == (72, 96) and db is None


def test_a_recorder_finds_them(oztt, fake):
    x, w, dy = fake(40, 96), fake(72, 96), fake(40, 72)
    assert "ops.oztt.linear.default" in make_fx(lambda *a: oztt.linear(*a, activation="gelu"))(x, w).code
    assert "ops.oztt.linear_backward.default" in make_fx(lambda *a: oztt.linear_backward(*a)[1])(dy, x, w).code


def test_activations_are_checked(oztt, fake):
    with pytest.raises(ValueError):
        oztt.linear(fake(4, 8), fake(8, 8), activation="tanh")
