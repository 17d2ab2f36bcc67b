"""A product whose kernel gave up a wait is reported to the optimiser too."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["step", "moments"])
def test_a_product_that_gave_up_is_reported_to_the_optimiser(oztt, cuda, call):
    """Gradients of a product whose kernel gave up a wait are not applied."""
    p = torch.ones(300, device="cuda")
    opt = oztt.AdamW([p], state_bits=8)
    oztt.call("oztt_test_linear_error", 2)
    with pytest.raises(RuntimeError, match="gave up waiting"):
        opt.step([torch.ones(300, device="cuda")]) if call == "step" else opt.moments()
    assert opt.t == 0 and torch.equal(p, torch.ones_like(p)) and not bool(opt.m.any())
    opt.step([torch.ones(300, device="cuda")])
    assert opt.t == 1 and not torch.equal(p, torch.ones_like(p))
