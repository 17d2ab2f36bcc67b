"""A wait that gave up is reported to the device that it happened on, and to a program that has no further call."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_status(oztt, cuda):
    x = torch.ones(8, 64, device="cuda", dtype=torch.bfloat16)
    want = oztt.linear(x, x)
    torch.cuda.synchronize()
    oztt.layer_status()
    oztt.call("oztt_test_linear_error", 4)
    with pytest.raises(RuntimeError, match=r"gave up waiting \(code 4\)"):
        oztt.layer_status()
    oztt.layer_status()  # once
    assert torch.equal(oztt.linear(x, x), want)


def test_another_devices_error(oztt, cuda):
    """Device 5's error stays device 5's."""
    x = torch.ones(8, 64, device="cuda", dtype=torch.bfloat16)
    want = oztt.linear(x, x)
    oztt.call("oztt_test_device_error", 5, 2)
    assert torch.equal(oztt.linear(x, x), want)
    oztt.AdamW([torch.ones(8, device="cuda")]).step([torch.ones(8, device="cuda")])
    oztt.layer_status()
    with pytest.raises(RuntimeError, match="code 2"):
        oztt.layer_status(5)
    oztt.layer_status(5)
