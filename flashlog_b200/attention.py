"""The attention over relation operators: the head that makes its logits, and the weights made of them.

The models turn a hidden state into a logit for each of the n = 2R + 1
relation operators with a linear layer (src/model_DRUM_kernel_sp.py:99-110),
and the hops propagate by the softmax of those logits:

* linear: y = act(x W^T + bias) + residual, in one product with its epilogue;
* relation_weights: the softmax, with what a rule's body may contain built in:
  penalties for operators that the body has already, a bias per operator, and
  a mask of the operators that may follow the body's state (such as
  rules.first_operator_mask).

Everything runs in the library's kernels on the current stream, forward and
backward, and can be captured in a CUDA graph.
"""
from __future__ import annotations

import dataclasses

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
    dt, shape = x.dtype, x.shape
    if dt not in ops.FL_DTYPE:
        raise ValueError(f"linear takes float32, float16 or bfloat16 tensors, got {dt}")
    if weight.dim() != 2 or not shape or shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x [..., k] and weight [n, k], got {tuple(shape)} and {tuple(weight.shape)}")
    n, k = weight.shape
    if n == 0 or k == 0:
        raise ValueError("linear: weight must not be empty")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != n):
        raise ValueError(f"linear: bias must be [{n}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != shape[:-1] + (n,):
        raise ValueError(f"linear: residual must be {tuple(shape[:-1] + (n,))}, got {tuple(residual.shape)}")
    for t in (weight, bias, residual):
        if t is not None and t.dtype != dt:
            raise ValueError(f"linear: tensors of one dtype, got {dt} and {t.dtype}")
    flat = len(shape) == 2
    if not flat:
        x = x.reshape(-1, k)
        residual = None if residual is None else residual.reshape(-1, n)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        y = _Linear.apply(x, weight, bias, residual, act)
    else:
        y, _ = ops.linear_forward(x, weight, bias, residual, act)
    return y if flat else y.view(shape[:-1] + (n,))


class _RelationWeights(autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, mask, states, history, tau, repetition, frequency, presence):
        w = ops.relation_weights(logits, bias, mask, states, history, tau, repetition, frequency, presence)
        ctx.tau, ctx.repetition = tau, repetition
        # the history matters to the gradient through the sign of penalised logits only
        ctx.save_for_backward(w, logits, bias, history if repetition != 1.0 else None)
        return w

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        w, logits, bias, history = ctx.saved_tensors
        dz = db = None
        if w.numel() == 0:
            dz, db = torch.zeros_like(logits), None if bias is None else torch.zeros_like(bias)
        elif ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            dz, db = ops.relation_weights_backward(w, g, logits, bias, history, ctx.tau, ctx.repetition,
                                                   ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dz, db, None, None, None, None, None, None, None


def relation_weights(logits, *, tau: float = 1.0, mask=None, states=None, bias=None, history=None,
                     repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0):
    """The hops' weights, fp32 [..., n], from logits [..., n] (fp32, fp16 or bf16; 1 <= n <= 65536):

        u = z / repetition (z > 0) or z * repetition (z <= 0) for operators in the row's history, z otherwise
        u = u - frequency * count - presence * [count > 0] + bias
        w = softmax(u / tau) over the operators that the mask allows, 0 elsewhere

    history: int64 [..., H], H <= 65535, the operators used so far (entries outside [0, n), such as a padding of -1, do not
    count).  bias: [n] or the logits' shape, of their dtype.  mask: bool or uint8; with states (int64 [...]) a
    table [S, n] of what may follow each state, and a state outside [0, S) allows nothing; without states [n],
    or the logits' shape.  A row with nothing left gets weights 0 (it propagates nothing) and gradient 0.  Masked
    logits may hold anything, NaN included; a NaN or +inf that is not masked makes its row NaN.  Differentiable
    once, in logits and bias."""
    if logits.dim() < 1 or logits.dtype not in ops.FL_DTYPE:
        raise ValueError(f"relation_weights takes float32, float16 or bfloat16 logits [..., n], got {logits.dtype}")
    lead, n = logits.shape[:-1], logits.shape[-1]
    if not 1 <= n <= ops.MAX_WEIGHT_COLUMNS:
        raise ValueError(f"relation_weights: need 1 to {ops.MAX_WEIGHT_COLUMNS} operators, got {n}")
    tau, repetition, frequency, presence = float(tau), float(repetition), float(frequency), float(presence)
    # compared as the fp32 values that the kernels use
    if not (1e-30 < tau < 1e30 and 1e-30 < repetition < 1e30):
        raise ValueError(f"relation_weights: tau and repetition must be positive, got {tau} and {repetition}")
    if not (abs(frequency) < 1e30 and abs(presence) < 1e30):
        raise ValueError(f"relation_weights: penalties must be finite, got {frequency} and {presence}")
    if bias is not None:
        if bias.dtype != logits.dtype or bias.shape not in ((n,), logits.shape):
            raise ValueError(f"relation_weights: bias must be [{n}] or the logits' shape, of their dtype")
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"relation_weights: mask must be bool or uint8, got {mask.dtype}")
        if states is not None:
            ok = mask.dim() == 2 and mask.shape[1] == n and mask.shape[0] > 0
        else:
            ok = mask.shape in ((n,), logits.shape)
        if not ok:
            raise ValueError(f"relation_weights: mask must be [states, {n}] with states, else [{n}] or the logits' "
                             f"shape, got {tuple(mask.shape)}")
    if states is not None and (mask is None or states.dtype != torch.int64 or states.shape != lead):
        raise ValueError(f"relation_weights: states must be int64 {tuple(lead)}, next to a mask")
    if history is not None and (history.dtype != torch.int64 or history.dim() < 1 or history.shape[:-1] != lead):
        raise ValueError(f"relation_weights: history must be int64 {tuple(lead)} + [H]")
    if history is not None and history.shape[-1] > ops.MAX_HISTORY:
        raise ValueError(f"relation_weights: at most {ops.MAX_HISTORY} history entries, got {history.shape[-1]}")
    z = ops._lines(logits if logits.dim() == 2 else logits.reshape(-1, n))
    if bias is not None:
        bias = bias.contiguous() if bias.dim() == 1 else bias.reshape(-1, n).contiguous()
    if mask is not None:
        mask = ops._lines(mask if mask.dim() == 2 else mask.reshape(-1, n))
    if states is not None:
        states = (states if states.dim() == 1 else states.reshape(-1)).contiguous()
    if history is not None:
        width = history.shape[-1]
        history = None if width == 0 else ops._lines(history if history.dim() == 2 else history.reshape(-1, width))
    if torch.is_grad_enabled() and (z.requires_grad or (bias is not None and bias.requires_grad)):
        w = _RelationWeights.apply(z, bias, mask, states, history, tau, repetition, frequency, presence)
    else:
        w = ops.relation_weights(z, bias, mask, states, history, tau, repetition, frequency, presence)
    return w if logits.dim() == 2 else w.view(logits.shape)


@dataclasses.dataclass
class OperatorRules:
    """What the attention of T hops may take, for engine.drum_propagate and
    step.DrumTrainStep (relation_weights applied to every query's channels):

    mask    bool or uint8 [S, n] with states int64 [T, Q]: the operators
            allowed in each state, and each query's state at each hop
    history int64 [Q, H]: operators that count as used (such as the query's
            own relation, to keep it out of its own rule)
    bias    [n], added to every query's logits
    repetition, frequency, presence: the penalties of used operators

    The step reads these tensors on every run: a captured step follows
    changes made to them in place."""

    mask: torch.Tensor | None = None
    states: torch.Tensor | None = None
    history: torch.Tensor | None = None
    bias: torch.Tensor | None = None
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0

    def check(self, T: int, Q: int, n: int):
        """Raise unless the tensors fit T hops of Q queries and n operators."""
        if (self.mask is None) != (self.states is None):
            raise ValueError("operator rules: mask and states come together")
        if self.mask is not None:
            if self.mask.dim() != 2 or self.mask.shape[1] != n or self.mask.dtype not in (torch.bool, torch.uint8):
                raise ValueError(f"operator rules: mask must be bool or uint8 [states, {n}]")
            if tuple(self.states.shape) != (T, Q) or self.states.dtype != torch.int64:
                raise ValueError(f"operator rules: states must be int64 [{T}, {Q}]")
        if self.history is not None and (self.history.dim() != 2 or self.history.shape[0] != Q or
                                         self.history.dtype != torch.int64):
            raise ValueError(f"operator rules: history must be int64 [{Q}, H]")
        if self.history is not None and self.history.shape[1] > ops.MAX_HISTORY:
            raise ValueError(f"operator rules: at most {ops.MAX_HISTORY} history entries")
        if self.bias is not None and (tuple(self.bias.shape) != (n,) or self.bias.dtype != torch.float32):
            raise ValueError(f"operator rules: bias must be float32 [{n}]")
        if not (1e-30 < self.repetition < 1e30 and abs(self.frequency) < 1e30 and abs(self.presence) < 1e30):
            raise ValueError("operator rules: repetition must be positive and the penalties finite")

    def rows(self, t: int, N: int):
        """Keyword arguments of relation_weights for hop t's rows r = q * N + channel."""
        kw = dict(repetition=self.repetition, frequency=self.frequency, presence=self.presence)
        if self.mask is not None:
            kw["mask"] = ops._lines(self.mask)
            kw["states"] = self.states[t][:, None].expand(-1, N).reshape(-1)
        if self.history is not None and self.history.shape[1] > 0:
            kw["history"] = self.history[:, None, :].expand(-1, N, -1).reshape(-1, self.history.shape[1])
        if self.bias is not None:
            kw["bias"] = self.bias.contiguous()
        return kw
