"""Orthogonalised updates (Muon) for the matrices that training learns.

The attention table [2R, T, N, n] is T N matrices from query relations to
operators, and a head's weight is one matrix.  The Muon step replaces the
plain SGD update of such a matrix by an update whose singular values are all
brought near 1 by Newton-Schulz products:

* orthogonalize: the products alone, for a batch of matrices;
* muon_update, muon_update_: momentum, orthogonalisation, weight decay and
  update of a parameter, into new tensors or in place;
* Muon: a torch optimizer around it.

step.DrumTrainStep(optimizer="muon") updates the attention table this way.
Everything runs in the library's kernels on the current stream and can be
captured in a CUDA graph.
"""
from __future__ import annotations

import math

import torch

from . import ops
from ._lib import bind

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _check(what, steps, coefficients, eps):
    if int(steps) != steps or not 1 <= steps <= 64:
        raise ValueError(f"{what}: 1 to 64 steps, got {steps}")
    c = tuple(float(v) for v in coefficients)
    if len(c) != 3 or not all(math.isfinite(v) for v in c):
        raise ValueError(f"{what}: three finite coefficients, got {coefficients}")
    eps = float(eps)
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError(f"{what}: eps must be finite and at least 0, got {eps}")
    return int(steps), c, eps


def _check_matrix(what, t):
    if t.dim() < 2 or t.shape[-1] == 0 or t.shape[-2] == 0:
        raise ValueError(f"{what} takes matrices [..., m, n], got {tuple(t.shape)}")


@torch.no_grad()
def orthogonalize(update, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
    """Newton-Schulz of each matrix of update [..., m, n] (fp32, fp16 or bf16):
    X = U / (|U|_F + eps), then `steps` times X <- a X + (b A + c A^2) X with
    A = X X^T of the shorter side.  Every matrix on the way keeps 22 bits and
    every product fp32 sums whatever the dtype, so the result is about as near
    as plain fp32 steps come, for decaying singular values too; it has the
    update's dtype and is rounded once.  Sides are below 2^24; of matrices too
    large for one block (from some 55 x 55 on) a batch has at most 65,535.  The
    coefficients must keep singular values of [0, 1] within 3.  A matrix that
    holds a NaN or an infinity gives NaN.  Not differentiable."""
    if update.dtype not in ops.FL_DTYPE:
        raise ValueError(f"orthogonalize takes float32, float16 or bfloat16 matrices, got {update.dtype}")
    _check_matrix("orthogonalize", update)
    steps, coefficients, eps = _check("orthogonalize", steps, coefficients, eps)
    return bind().orthogonalize(update, steps, coefficients, eps)


def _check_gate(gate):
    if gate is not None and (gate.dtype != torch.float32 or gate.numel() != 1):
        raise ValueError("muon_update: gate must be one float32")


def _muon_args(param, grad, momentum, lr, beta, nesterov, weight_decay, scale, steps, coefficients, eps):
    _check_matrix("muon_update", param)
    for name, t in (("param", param), ("grad", grad), ("momentum", momentum)):
        if t.dtype != torch.float32 or t.shape != param.shape:
            raise ValueError(f"muon_update: {name} must be float32 {tuple(param.shape)}, got {t.dtype} "
                             f"{tuple(t.shape)}")
    steps, coefficients, eps = _check("muon_update", steps, coefficients, eps)
    lr, beta, weight_decay = float(lr), float(beta), float(weight_decay)
    if not all(math.isfinite(v) for v in (lr, weight_decay)) or not 0.0 <= beta < 1.0:
        raise ValueError(f"muon_update: lr and weight_decay must be finite and 0 <= beta < 1, got {lr}, "
                         f"{weight_decay} and {beta}")
    m, n = param.shape[-2:]
    scale = math.sqrt(max(1.0, m / n)) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"muon_update: scale must be finite, got {scale}")
    return lr, beta, bool(nesterov), weight_decay, scale, steps, coefficients, eps


def _overlaps_itself(t):
    """Whether two elements of t may share memory (an expanded or overlapping view)."""
    dims = sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1)
    reach = 0
    for s, n in dims:
        if s <= reach:
            return True
        reach += s * (n - 1)
    return False


def _range(t):
    first = t.data_ptr()
    return first, first + t.element_size() * (1 + sum(s * (n - 1) for n, s in zip(t.shape, t.stride())))


@torch.no_grad()
def muon_update(param, grad, momentum, *, lr: float, beta: float = 0.95, nesterov: bool = True,
                weight_decay: float = 0.0, scale=None, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
                gate=None):
    """One Muon step of param [..., m, n] (a batch of matrices), all fp32:

        momentum' = beta * momentum + grad;  U = grad + beta * momentum' (nesterov) or momentum'
        param' = param * (1 - lr * weight_decay) - lr * scale * orthogonalize(U)

    scale defaults to sqrt(max(1, m / n)).  gate (a float32 on the device): where it holds 0 -- a step that
    failed, found on the device -- both come out as they went in.  Returns (param', momentum') as new tensors."""
    _check_gate(gate)
    args = _muon_args(param, grad, momentum, lr, beta, nesterov, weight_decay, scale, steps, coefficients, eps)
    p2, m2 = torch.empty_like(param), torch.empty_like(momentum)
    bind().muon_update(param, grad, momentum, p2, m2, *args, gate)
    return p2, m2


@torch.no_grad()
def muon_update_(param, grad, momentum, *, lr: float, beta: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, scale=None, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
                 gate=None):
    """muon_update in place: param and momentum are overwritten; returns param.  param, grad and momentum must lie
    apart in memory."""
    _check_gate(gate)
    args = _muon_args(param, grad, momentum, lr, beta, nesterov, weight_decay, scale, steps, coefficients, eps)
    if _overlaps_itself(param) or _overlaps_itself(momentum):
        raise ValueError("muon_update_: param and momentum must not overlap themselves")
    spans = sorted(_range(t) for t in (param, grad, momentum)) if param.numel() else []
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("muon_update_: param, grad and momentum must lie apart in memory")
    bind().muon_update(param, grad, momentum, param, momentum, *args, gate)
    return param


class Muon(torch.optim.Optimizer):
    """muon_update_ for every parameter, as a torch optimizer.  Parameters are
    fp32 with at least two dimensions; the last two are the matrix (a table
    [2R, T, N, n] trained as T N matrices goes in as table.permute(1, 2, 0, 3),
    a leaf of that shape).  Parameters without a gradient are left alone."""

    def __init__(self, params, lr: float = 0.02, beta: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, scale=None, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
        super().__init__(params, dict(lr=lr, beta=beta, nesterov=nesterov, weight_decay=weight_decay, scale=scale,
                                      steps=steps, coefficients=tuple(coefficients), eps=eps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dtype != torch.float32 or p.dim() < 2:
                    raise ValueError(f"Muon takes float32 parameters of at least two dimensions, got {p.dtype} "
                                     f"{tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            args = {k: v for k, v in group.items() if k != "params"}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("Muon does not take sparse gradients")
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p)
                muon_update_(p, p.grad, state["momentum"], **args)
        return loss
