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

from . import _lib as L
from . import ops
from ._lib import bind

ACTIVATIONS = {"none": L.FL_ACT_NONE, "relu": L.FL_ACT_RELU, "tanh": L.FL_ACT_TANH, "silu": L.FL_ACT_SILU,
               "gelu": L.FL_ACT_GELU}


def linear(x, weight, bias=None, residual=None, activation: str = "none"):
    """act(x W^T + bias) + residual: x [..., k], weight [n, k], bias [n],
    residual [..., n], all fp32, fp16 or bf16 on one CUDA device; the result
    [..., n] has their dtype.  activation: none, relu, tanh, silu or gelu (the
    erf form).  Differentiable once in every tensor.

    Sums run in fp32 whatever the dtype.  fp32 values keep 22 bits or more down
    to 2^-29 of the largest of their row (of x or weight; in the backward also
    of their column), and are off by at most 2^-50 of that below.  A fp32 row
    (or weight row) that holds an infinity gives NaN.  A backward pass takes at
    most 8,388,480 rows."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return bind().linear(x, weight, bias, residual, act)


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
    return bind().relation_weights(logits, tau, mask, states, bias, history, repetition, frequency, presence)


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

    def rows(self, t: int, N: int, history=None):
        """Keyword arguments of relation_weights for hop t's rows r = q * N + channel.  history: the queries' histories
        by row, where the caller has them (they are the same for every hop)."""
        kw = dict(repetition=self.repetition, frequency=self.frequency, presence=self.presence)
        if self.mask is not None:
            kw["mask"] = ops._lines(self.mask)
            kw["states"] = self.states[t][:, None].expand(-1, N).reshape(-1)
        if history is not None:
            kw["history"] = history
        elif self.history is not None and self.history.shape[1] > 0:
            kw["history"] = self.history[:, None, :].expand(-1, N, -1).reshape(-1, self.history.shape[1])
        if self.bias is not None:
            kw["bias"] = self.bias.contiguous()
        return kw
