"""What the optimiser steps is another version of its tensor, whoever asked for gradients when."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["detached", "later", "leaf", "master"])
def test_a_graph_over_old_weights_is_noticed(oztt, cuda, how):
    """A backward pass over what was saved before the step runs into torch's check of versions."""
    leaf = torch.randn(500, device="cuda", requires_grad=how != "later")
    given = {"detached": leaf.detach(), "later": leaf, "leaf": leaf, "master": leaf.detach().bfloat16()}[how]
    opt = oztt.AdamW([given], masters=[leaf.detach()] if how == "master" else None)
    if how == "later":
        leaf.requires_grad_(True)
    y = (leaf * leaf).sum()
    opt.step([torch.ones(500, device="cuda")])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_parameter_without_a_gradient_keeps_its_version(oztt, cuda):
    p, q = (torch.ones(10, device="cuda") for _ in range(2))
    opt = oztt.AdamW([p, q])
    before = p._version, q._version
    opt.step([None, torch.ones(10, device="cuda")])
    assert p._version == before[0] and q._version > before[1]
