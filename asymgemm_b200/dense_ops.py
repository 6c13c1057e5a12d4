"""Dense product with bias, activation and residual in its epilogue, and its gradients (csrc/dense.cu): what an MoE layer needs
besides its experts -- router logits, shared experts, projections -- with the weights in device memory. (Weights in pinned host
memory are the grouped GEMMs' business: a single dense product would read them at the host link's rate.)

The kernels are tcgen05 products fed by TMA, so rows of `x` and `weight` start on 16-byte boundaries: k is a multiple of 8.
Everything runs on the current stream; there is no CPU branch. `linear` is recorded by autograd; `linear_backward` is the same
gradient as a function of its own, which is the form to capture into a CUDA graph. Forward-mode derivatives are refused.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib, api

_ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _activation(name: str) -> int:
    if name not in _ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {', '.join(map(repr, _ACTIVATIONS))}, got {name!r}")
    return _ACTIVATIONS[name]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
           return_pre: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, Optional[torch.Tensor]]]:
    """y = act(x weight^T + bias) + residual in one kernel: x [..., k], weight [n, k] (both bf16 or both fp16), bias [n] (their type or
    fp32), residual [..., n] (type of the output) -> y [..., n] in `out_dtype`: the operands' type (default) or torch.float32.
    `activation`: "none", "relu", "gelu" (x Phi(x)) or "silu". x, weight and residual may have any distance between rows (rows that
    lie on one another, as in an expanded tensor, are copied out first).

    Sums are fp32, rounded once to the output's type. (fp32 outputs, e.g. router logits, are off by 4.5e-7 of their norm at k = 7168,
    where an fp32 product of the same operands is by 1.4e-7 to 9e-7.) `return_pre`: also return z = x weight^T + bias in the operands' type, which `linear_backward` needs
    for an activation (None without one). Differentiable with respect to x, weight, bias and residual."""
    api._refuse_tangents(x, weight, bias, residual)
    act = _activation(activation)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype != x.dtype and out_dtype != torch.float32:
        raise RuntimeError("out_dtype must be x's type or torch.float32")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        y, pre = _Linear.apply(x, weight, bias, residual, act, out_dtype)
    else:
        y, pre = _forward(x, weight, bias, residual, act, out_dtype, return_pre)
    return (y, pre) if return_pre else y


def _forward(x, weight, bias, residual, act, out_dtype, keep_pre):
    flat = x.dim() == 2
    if not flat:
        shape = x.shape[:-1] + (weight.shape[0],)
        if x.dim() == 0 or (residual is not None and residual.shape != shape):
            raise RuntimeError("x is [..., k] and residual [..., n] with the same leading dimensions")
        x = x.reshape(-1, x.shape[-1])
        residual = residual.reshape(-1, residual.shape[-1]) if residual is not None else None
    y, pre = _lib.torch_ops().linear(x, weight, bias, act, residual, out_dtype == torch.float32, bool(keep_pre and act != 0),
                                     api._status_word(x.device), api._state["timeout_ms"])
    if flat:
        return y, pre
    return y.view(shape), pre.view(shape) if pre is not None else None


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, activation: str = "none", pre: Optional[torch.Tensor] = None,
                    need_x: bool = True, need_weight: bool = True, need_bias: bool = True,
                    bias_dtype: Optional[torch.dtype] = None) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients of `linear` from dy [..., n] (the operands' type or fp32): (dx like x, dweight like weight, dbias [n] in `bias_dtype`:
    the operands' type (default) or fp32), None for one that is not needed. `pre`: what `linear(..., return_pre=True)` returned,
    for an activation. The gradient of the residual is dy.

    dz = dy act'(z) is rounded to the operands' type (as dy is where it is fp32) because the tensor cores take it as an operand;
    dbias sums it before that rounding, in fp32 and in a fixed order."""
    api._refuse_tangents(dy, x, weight, pre)
    act = _activation(activation)
    bias_dtype = x.dtype if bias_dtype is None else bias_dtype
    if bias_dtype != x.dtype and bias_dtype != torch.float32:
        raise RuntimeError("bias_dtype must be x's type or torch.float32")
    shape = x.shape
    if x.dim() != 2:
        if x.dim() == 0 or dy.shape[:-1] != shape[:-1]:
            raise RuntimeError("x is [..., k] and dy [..., n] with the same leading dimensions")
        x, dy = x.reshape(-1, shape[-1]), dy.reshape(-1, dy.shape[-1])
        pre = pre.reshape(-1, pre.shape[-1]) if pre is not None else None
    dx, dweight, dbias = _lib.torch_ops().linear_backward(dy, x, weight, act, pre, bool(need_x), bool(need_weight), bool(need_bias),
                                                          bias_dtype == torch.float32, api._status_word(x.device), api._state["timeout_ms"])
    return dx.view(shape) if dx is not None else None, dweight, dbias


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_dtype):
        y, pre = _forward(x, weight, bias, residual, act, out_dtype, True)
        ctx.save_for_backward(x, weight, pre)
        ctx.act = next(name for name, code in _ACTIVATIONS.items() if code == act)
        ctx.bias_dtype = bias.dtype if bias is not None else None
        if pre is not None:
            ctx.mark_non_differentiable(pre)
        return y, pre

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, weight, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dweight = dbias = None
        if any(need[:3]):
            rows = dy if dy.stride(-1) == 1 or dy.shape[-1] == 1 else dy.contiguous()
            dx, dweight, dbias = linear_backward(rows, x, weight, ctx.act, pre, need[0], need[1], need[2], ctx.bias_dtype)
        return dx, dweight, dbias, dy if need[3] else None, None, None
