"""The product of a network layer with bias, activation and residual in its epilogue, and its gradients, on CUDA
tensors of torch (oztt_linear_forward and oztt_linear_backward of the C ABI).

BF16 or FP16 throughout; sums in 32 bits, every result rounded once. The calls run on the current stream of the
tensors' device and do not wait for it. No counterpart in the reference, whose products are FP64 only.
"""

from __future__ import annotations

import torch

from . import _binding

__all__ = ["ACTIVATIONS", "linear", "linear_backward"]

# OZTT_ACT_* of include/oztt_cuda.h
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}

_torch = _binding()  # csrc/torch_binding.cpp: the checks, the results' tensors, the current stream


def _activation(who: str, activation: str) -> int:
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"{who}: activation must be one of {', '.join(ACTIVATIONS)}, not {activation!r}")
    return act


# The same calls as operators of torch's dispatcher, for those that have to go through it (a tracer or another recorder,
# tensors without memory): results that were not asked for are empty tensors there.


@torch.library.custom_op("oztt::linear", mutates_args=())
def _dispatched_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None,
                       activation: str, save_pre: bool) -> tuple[torch.Tensor, torch.Tensor]:
    y, pre = _torch.linear(x, weight, bias, residual, ACTIVATIONS[activation], save_pre, False)
    return y, pre if save_pre else x.new_empty(0)


@_dispatched_linear.register_fake
def _(x, weight, bias, residual, activation, save_pre):
    y = x.new_empty((*x.shape[:-1], weight.shape[0]))
    return y, torch.empty_like(y) if save_pre else x.new_empty(0)


@torch.library.custom_op("oztt::linear_backward", mutates_args=())
def _dispatched_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, pre: torch.Tensor | None,
                         activation: str, need_input: bool, need_weight: bool,
                         need_bias: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    out = _torch.linear_backward(dy, x, weight, pre, ACTIVATIONS[activation], need_input, need_weight, need_bias, False)
    return tuple(dy.new_empty(0) if t is None else t for t in out)


@_dispatched_backward.register_fake
def _(dy, x, weight, pre, activation, need_input, need_weight, need_bias):
    return (dy.new_empty(x.shape if need_input else 0), dy.new_empty(weight.shape if need_weight else 0),
            dy.new_empty(weight.shape[0] if need_bias else 0))


def _keep(ctx, inputs, output):
    x, weight, _, _, activation, _ = inputs
    ctx.save_for_backward(x, weight, output[1] if activation != "none" else None)
    ctx.activation = activation
    ctx.mark_non_differentiable(output[1])


def _gradients(ctx, dy, _):
    x, weight, pre = ctx.saved_tensors
    need = ctx.needs_input_grad
    out = _dispatched_backward(dy, x, weight, pre, ctx.activation, *need[:3])
    return (*(g if n else None for g, n in zip(out, need)), dy if need[3] else None, None, None)


_dispatched_linear.register_autograd(_gradients, setup_context=_keep)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, save_pre):
        keep = save_pre or activation != "none"
        y, pre = _torch.linear(x, weight, bias, residual, ACTIVATIONS[activation], keep, False)
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
    the activation, which linear_backward needs for one. Differentiable with respect to all four tensors, once and in
    reverse mode: tangents of the forward mode and torch.func's transforms are refused with RuntimeError.
    Raises ValueError for what does not fit together, RuntimeError for a CUDA failure, torch.OutOfMemoryError where the
    result or the call's scratch memory, both from torch's allocator, finds no room."""
    out = _torch.linear(x, weight, bias, residual, _activation("linear", activation), bool(save_pre), True)
    if out is None:  # a gradient is wanted
        out = _Linear.apply(x, weight, bias, residual, activation, bool(save_pre))
    elif out is NotImplemented:
        wanted = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))
        out = _dispatched_linear(x, weight, bias, residual, activation, bool(save_pre) or (wanted and activation != "none"))
    return out if save_pre else out[0]


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, *, pre: torch.Tensor | None = None,
                    activation: str = "none", need_input: bool = True, need_weight: bool = True,
                    need_bias: bool = True):
    """The gradients (dx, dweight, dbias) of linear for the gradient dy [..., n] of its output; those not needed are
    None. pre [..., n], linear's second result, is needed with an activation. The gradient of the residual is dy.
    dy act'(pre) is rounded to the tensors' type once before the products, not before the sum for dbias. The results
    carry no gradients of their own; forward-mode tangents are refused with RuntimeError."""
    need = bool(need_input), bool(need_weight), bool(need_bias)
    out = _torch.linear_backward(dy, x, weight, pre, _activation("linear_backward", activation), *need, True)
    if out is NotImplemented:
        out = tuple(g if n else None for g, n in zip(_dispatched_backward(dy, x, weight, pre, activation, *need), need))
    return out
