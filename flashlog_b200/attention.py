"""The attention over relation operators: the head that makes its logits.

The models turn a hidden state into a logit for each of the n = 2R + 1
relation operators with a linear layer (src/model_DRUM_kernel_sp.py:99-110),
and the hops propagate by the softmax of those logits:

* linear: y = act(x W^T + bias) + residual, in one product with its epilogue.

Everything runs in the library's kernels on the current stream, forward and
backward, and can be captured in a CUDA graph.
"""
from __future__ import annotations

import torch
from torch import autograd
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import ops

ACTIVATIONS = {"none": L.FL_ACT_NONE, "relu": L.FL_ACT_RELU, "tanh": L.FL_ACT_TANH, "silu": L.FL_ACT_SILU,
               "gelu": L.FL_ACT_GELU}


class _Linear(autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, z = ops.linear_forward(x, weight, bias, residual, act, want_z=True)
        ctx.act, ctx.has_bias = act, bias is not None
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, weight, z = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx = dw = db = None
        if want[0] or want[1] or want[2]:
            dx, dw, db = ops.linear_backward(x, weight, z, gy, ctx.act, want[:3])
        return dx, dw, db, gy if want[3] else None, None


def linear(x, weight, bias=None, residual=None, activation: str = "none"):
    """act(x W^T + bias) + residual: x [..., k], weight [n, k], bias [n],
    residual [..., n], all fp32, fp16 or bf16 on one CUDA device; the result
    [..., n] has their dtype.  activation: none, relu, tanh, silu or gelu (the
    erf form).  Differentiable once in every tensor.

    Sums run in fp32 whatever the dtype; fp32 keeps fp32 accuracy.  A fp32 row
    (or weight row) that holds an infinity gives NaN."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    dt = x.dtype
    if dt not in ops.FL_DTYPE:
        raise ValueError(f"linear takes float32, float16 or bfloat16 tensors, got {dt}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x [..., k] and weight [n, k], got {tuple(x.shape)} and {tuple(weight.shape)}")
    n, k = weight.shape
    if n == 0 or k == 0:
        raise ValueError("linear: weight must not be empty")
    shape = x.shape[:-1] + (n,)
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"linear: bias must be [{n}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"linear: residual must be {tuple(shape)}, got {tuple(residual.shape)}")
    for t in (weight, bias, residual):
        if t is not None and t.dtype != dt:
            raise ValueError(f"linear: tensors of one dtype, got {dt} and {t.dtype}")
    ops._one_device("linear", x, weight, bias, residual)
    if x.dim() != 2:
        x = x.reshape(-1, k)
        residual = None if residual is None else residual.reshape(-1, n)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        y = _Linear.apply(x, weight, bias, residual, act)
    else:
        y, _ = ops.linear_forward(x, weight, bias, residual, act)
    return y if len(shape) == 2 else y.view(shape)
