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
    reverse mode: a tangent of the forward mode is refused with RuntimeError.
    Raises ValueError for what does not fit together, RuntimeError for a CUDA failure."""
    out = _torch.linear(x, weight, bias, residual, _activation("linear", activation), bool(save_pre), True)
    if out is None:  # a gradient is wanted
        out = _Linear.apply(x, weight, bias, residual, activation, bool(save_pre))
    return out if save_pre else out[0]


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, *, pre: torch.Tensor | None = None,
                    activation: str = "none", need_input: bool = True, need_weight: bool = True,
                    need_bias: bool = True):
    """The gradients (dx, dweight, dbias) of linear for the gradient dy [..., n] of its output; those not needed are
    None. pre [..., n], linear's second result, is needed with an activation. The gradient of the residual is dy.
    dy act'(pre) is rounded to the tensors' type once before the products, not before the sum for dbias. The results
    carry no gradients of their own; forward-mode tangents are refused with RuntimeError."""
    return _torch.linear_backward(dy, x, weight, pre, _activation("linear_backward", activation), bool(need_input),
                                  bool(need_weight), bool(need_bias))
