"""The product of a network layer with bias, activation and residual in its epilogue, and its gradients, on CUDA
tensors of torch (oztt_linear_forward and oztt_linear_backward of the C ABI).

BF16 or FP16 throughout; sums in 32 bits, every result rounded once. The calls run on the current stream of the
tensors' device and do not wait for it. No counterpart in the reference, whose products are FP64 only.
"""

from __future__ import annotations

import struct
import threading

import torch

from . import OK, Format, _errbuf, _lib, _raise

__all__ = ["ACTIVATIONS", "linear", "linear_backward"]

# OZTT_ACT_* of include/oztt_cuda.h
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_FORMATS = {torch.bfloat16: int(Format.BF16), torch.float16: int(Format.FP16)}

_FORWARD = struct.Struct("=ii3Q" + 6 * "Qqq")   # oztt_linear
_BACKWARD = struct.Struct("=ii3Q" + 7 * "Qqq")  # oztt_linear_grad

_thread = threading.local()


def _error_buffer():
    try:
        return _thread.err
    except AttributeError:
        _thread.err = _errbuf()
        return _thread.err


def _call(name: str, device: torch.device, args: bytes) -> None:
    err = _error_buffer()
    rc = getattr(_lib(), name)(device.index, args, torch._C._cuda_getCurrentRawStream(device.index), err, 1024)
    if rc != OK:
        _raise(rc, err.value)


def _view(t: torch.Tensor | None) -> tuple[int, int, int]:
    """oztt_view of a matrix (or a vector, as one row)."""
    if t is None:
        return 0, 0, 0
    s = t.stride()
    return (t.data_ptr(), s[0], s[1]) if len(s) == 2 else (t.data_ptr(), 0, s[0])


def _check(who: str, first: torch.Tensor, **tensors: torch.Tensor | None) -> int:
    """The tensors' common format; ValueError for what cannot be computed with."""
    dtype, device = first.dtype, first.device
    if device.type != "cuda":
        raise ValueError(f"{who}: the tensors must be on a CUDA device")
    fmt = _FORMATS.get(dtype)
    if fmt is None:
        raise ValueError(f"{who}: the type must be torch.bfloat16 or torch.float16, not {dtype}")
    for name, t in tensors.items():
        if t is not None and (t.dtype != dtype or t.device != device):
            raise ValueError(f"{who}: {name} is {t.dtype} on {t.device}, not {dtype} on {device}")
    return fmt


def _activation(who: str, activation: str) -> int:
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"{who}: activation must be one of {', '.join(ACTIVATIONS)}, not {activation!r}")
    return act


def _forward(x, weight, bias, residual, activation, save_pre):
    fmt = _check("linear", x, weight=weight, bias=bias, residual=residual)
    act = _activation("linear", activation)
    shape = x.shape
    if weight.dim() != 2 or not shape or shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x {tuple(shape)} does not match weight {tuple(weight.shape)}")
    n, k = weight.shape
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != n):
        raise ValueError(f"linear: bias {tuple(bias.shape)} does not match weight {tuple(weight.shape)}")
    out_shape = shape[:-1] + (n,)
    if residual is not None and residual.shape != out_shape:
        raise ValueError(f"linear: residual {tuple(residual.shape)} does not match the output {tuple(out_shape)}")
    flat = len(shape) != 2
    if flat:
        m = 1
        for d in shape[:-1]:
            m *= d
        x = x.reshape(m, k)
        residual = residual.reshape(m, n) if residual is not None else None
    else:
        m = shape[0]
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    pre = torch.empty((m, n), dtype=x.dtype, device=x.device) if save_pre else None
    _call("oztt_linear_forward", x.device,
          _FORWARD.pack(fmt, act, m, n, k, *_view(x), *_view(weight), *_view(bias), *_view(residual), y.data_ptr(), n,
                        1, pre.data_ptr() if save_pre else 0, n, 1))
    if flat:
        y = y.view(out_shape)
        pre = pre.view(out_shape) if save_pre else None
    return y, pre


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, save_pre):
        keep = save_pre or activation != "none"
        y, pre = _forward(x, weight, bias, residual, activation, keep)
        ctx.save_for_backward(x, weight, pre if activation != "none" else None)
        ctx.activation = activation
        if save_pre:
            ctx.mark_non_differentiable(pre)
        return y, (pre if save_pre else None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, weight, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = linear_backward(dy, x, weight, pre=pre, activation=ctx.activation, need_input=need[0],
                                     need_weight=need[1], need_bias=need[2])
        return dx, dw, db, dy if need[3] else None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           residual: torch.Tensor | None = None, activation: str = "none", save_pre: bool = False):
    """act(x weight^T + bias) + residual.

    x [..., k], weight [n, k], bias [n], residual [..., n], all BF16 or all FP16 on one CUDA device, any strides
    (a weight stored as [k, n] is passed as its transpose). activation: "none", "relu", "gelu" (with the error
    function), "gelu_tanh" or "silu". Returns y [..., n], or with save_pre (y, pre), pre = x weight^T + bias before
    the activation, which linear_backward needs for one. Differentiable with respect to all four tensors.
    Raises ValueError for what does not fit together, RuntimeError for a CUDA failure."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        y, pre = _Linear.apply(x, weight, bias, residual, activation, save_pre)
    else:
        y, pre = _forward(x, weight, bias, residual, activation, save_pre)
    return (y, pre) if save_pre else y


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, *, pre: torch.Tensor | None = None,
                    activation: str = "none", need_input: bool = True, need_weight: bool = True,
                    need_bias: bool = True):
    """The gradients (dx, dweight, dbias) of linear for the gradient dy [..., n] of its output; those not needed are
    None. pre [..., n], linear's second result, is needed with an activation. The gradient of the residual is dy.
    dy act'(pre) is rounded to the tensors' type once before the products, not before the sum for dbias."""
    fmt = _check("linear_backward", dy, x=x, weight=weight, pre=pre)
    act = _activation("linear_backward", activation)
    if weight.dim() != 2 or not x.dim() or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_backward: x {tuple(x.shape)} does not match weight {tuple(weight.shape)}")
    n, k = weight.shape
    if dy.shape != x.shape[:-1] + (n,):
        raise ValueError(f"linear_backward: dy {tuple(dy.shape)} does not match x {tuple(x.shape)} and weight "
                         f"{tuple(weight.shape)}")
    if act and pre is None:
        raise ValueError(f"linear_backward: activation {activation!r} needs pre")
    if pre is not None and pre.shape != dy.shape:
        raise ValueError(f"linear_backward: pre {tuple(pre.shape)} does not match dy {tuple(dy.shape)}")
    shape = x.shape
    if len(shape) != 2:
        m = 1
        for d in shape[:-1]:
            m *= d
        x, dy = x.reshape(m, k), dy.reshape(m, n)
        pre = pre.reshape(m, n) if pre is not None else None
    else:
        m = shape[0]
    new = lambda *s: torch.empty(s, dtype=dy.dtype, device=dy.device)  # noqa: E731
    dx = new(m, k) if need_input else None
    dw = new(n, k) if need_weight else None
    db = new(n) if need_bias else None
    if need_input or need_weight or need_bias:
        _call("oztt_linear_backward", dy.device,
              _BACKWARD.pack(fmt, act, m, n, k, *_view(dy), *_view(pre), *_view(x), *_view(weight), *_view(dx),
                             *_view(dw), *_view(db)))
    return dx.view(shape) if need_input and len(shape) != 2 else dx, dw, db
