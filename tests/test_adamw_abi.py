"""Refusals of the AdamW step at the C ABI: checked on the host, before any device work."""

import struct

import pytest

TENSOR, MOMENTS, HYPER = struct.Struct("=4Q2i"), struct.Struct("=i4x4Q"), struct.Struct("=5dQQI4x")
GOOD_HYPER = (1e-3, 0.9, 0.999, 1e-8, 0.01, 1, 0, 0)


def step(oztt, tensors=((4096, 8192, 0, 10, 2, 2),), moments=(32, 4096, 8192, 0, 0), hyper=GOOD_HYPER, device=0):
    table = b"".join(TENSOR.pack(*t) for t in tensors)
    oztt.call("oztt_adamw_step", device, table, len(tensors), MOMENTS.pack(*moments), HYPER.pack(*hyper), None)


def changed(values, i, x):
    return values[:i] + (x,) + values[i + 1:]


@pytest.mark.parametrize("i,x,text", [(0, -1.0, "lr"), (0, float("nan"), "lr"), (0, float("inf"), "lr"), (1, 1.0, "betas"),
                                      (2, -0.5, "betas"), (2, float("nan"), "betas"), (3, -1e-9, "eps"),
                                      (4, float("inf"), "weight_decay"), (5, 0, "counted from 1"), (6, 4098, "grad_scale")])
def test_hyper_refusals(oztt, i, x, text):
    with pytest.raises(ValueError, match=text):
        step(oztt, hyper=changed(GOOD_HYPER, i, x))


@pytest.mark.parametrize("tensor,text", [((4096, 8192, 0, 10, 3, 2), "types"), ((4096, 8192, 0, 10, 2, -1), "types"),
                                         ((0, 8192, 0, 10, 2, 2), "missing"), ((4098, 8192, 0, 10, 2, 2), "aligned"),
                                         ((4096, 8193, 0, 10, 2, 0), "aligned"), ((4096, 8192, 4097, 10, 0, 0), "aligned"),
                                         ((4096, 8192, 0, 1 << 42, 2, 2), "too many")])
def test_tensor_refusals(oztt, tensor, text):
    with pytest.raises(ValueError, match=text):
        step(oztt, tensors=((4096, 8192, 0, 1, 2, 2), tensor))


@pytest.mark.parametrize("moments,text", [((16, 4096, 8192, 0, 0), "8 or 32"), ((32, 0, 8192, 0, 0), "missing"),
                                          ((8, 4096, 8192, 0, 4096), "missing"), ((32, 4100, 8192, 0, 0), "aligned")])
def test_moment_refusals(oztt, moments, text):
    with pytest.raises(ValueError, match=text):
        step(oztt, moments=moments)


def test_device_refusal(oztt):
    with pytest.raises(ValueError, match="device_id"):
        step(oztt, device=-1)


def test_nothing_to_do(oztt):
    step(oztt, tensors=())
    step(oztt, tensors=((0, 0, 0, 10, 2, 2), (4096, 8192, 0, 0, 2, 2)), moments=(8, 0, 0, 0, 0))
    oztt.call("oztt_adamw_values", 0, MOMENTS.pack(8, 0, 0, 0, 0), 0, None, None, None)


def test_values_refusals(oztt):
    with pytest.raises(ValueError, match="8-bit"):
        oztt.call("oztt_adamw_values", 0, MOMENTS.pack(32, 4096, 8192, 0, 0), 1, 4096, 8192, None)
    with pytest.raises(ValueError, match="outputs"):
        oztt.call("oztt_adamw_values", 0, MOMENTS.pack(8, 4096, 8192, 64, 64), 1, 0, 8192, None)
