"""Refusals of the layer products at the C ABI: checked on the host, before any device work."""

import struct

import pytest

FORWARD, BACKWARD = struct.Struct("=ii3Q" + 6 * "Qqq"), struct.Struct("=ii3Q" + 7 * "Qqq")
SOME = (4096, 8, 1)  # a view that a refused call never reads
NONE = (0, 0, 0)


def forward(oztt, fmt=0, act=0, m=4, n=4, k=8, x=SOME, w=SOME, b=NONE, r=NONE, y=SOME, pre=NONE, device=0):
    oztt.call("oztt_linear_forward", device, FORWARD.pack(fmt, act, m, n, k, *x, *w, *b, *r, *y, *pre), None)


def backward(oztt, fmt=0, act=0, m=4, n=4, k=8, dy=SOME, pre=NONE, x=SOME, w=SOME, dx=SOME, dw=SOME, db=NONE, device=0):
    oztt.call("oztt_linear_backward", device, BACKWARD.pack(fmt, act, m, n, k, *dy, *pre, *x, *w, *dx, *dw, *db), None)


@pytest.mark.parametrize("kw,text", [(dict(fmt=5), "BF16 or FP16"), (dict(fmt=2), "BF16 or FP16"),
                                     (dict(act=5), "activation"), (dict(act=-1), "activation"),
                                     (dict(x=NONE), "x is missing"), (dict(w=NONE), "w is missing"),
                                     (dict(y=NONE), "y is missing"), (dict(x=(4097, 8, 1)), "aligned"),
                                     (dict(w=(4096, -8, 1)), "negative"), (dict(b=(4096, 0, -1)), "negative"),
                                     (dict(y=(4096, 0, 1)), "must not be zero"), (dict(pre=(4096, 8, 0)), "must not be zero"),
                                     (dict(device=-1), "device_id")])
def test_forward_refusals(oztt, kw, text):
    with pytest.raises(ValueError, match=text):
        forward(oztt, **kw)


@pytest.mark.parametrize("kw,text", [(dict(fmt=4), "BF16 or FP16"), (dict(act=9), "activation"),
                                     (dict(act=2), "pre"), (dict(dy=NONE), "dy is missing"),
                                     (dict(x=NONE), "x is missing"), (dict(w=NONE), "w is missing"),
                                     (dict(dx=(4099, 8, 1)), "aligned"), (dict(dw=(4096, 0, 1)), "must not be zero"),
                                     (dict(db=(4096, 0, 0)), "must not be zero"), (dict(device=-3), "device_id")])
def test_backward_refusals(oztt, kw, text):
    with pytest.raises(ValueError, match=text):
        backward(oztt, **kw)


def test_nothing_to_do(oztt):
    forward(oztt, m=0, x=NONE, y=NONE)
    forward(oztt, n=0, w=NONE, y=NONE)


def test_no_arguments(oztt):
    for name in ("oztt_linear_forward", "oztt_linear_backward"):
        with pytest.raises(ValueError, match="no arguments"):
            oztt.call(name, 0, None, None)
