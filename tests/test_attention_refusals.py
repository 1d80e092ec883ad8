"""Calls that the attention operators refuse, before anything reaches a GPU (CPU tests)."""
import ctypes

import pytest
import torch

from flashlog_b200 import _lib as L
from flashlog_b200 import attention, muon
from flashlog_b200.step import DrumTrainStep

X, W = torch.zeros(3, 4), torch.zeros(5, 4)


@pytest.mark.parametrize("kw,message", [
    (dict(activation="swish"), "activation"),
    (dict(x=X.double(), weight=W.double()), "float32, float16 or bfloat16"),
    (dict(x=X.long(), weight=W.long()), "float32, float16 or bfloat16"),
    (dict(weight=W.half()), "one dtype"),
    (dict(weight=torch.zeros(5, 3)), r"x \[..., k\]"),
    (dict(weight=torch.zeros(4)), r"x \[..., k\]"),
    (dict(x=torch.zeros(())), r"x \[..., k\]"),
    (dict(weight=torch.zeros(0, 4)), "empty"),
    (dict(bias=torch.zeros(4)), "bias"),
    (dict(bias=torch.zeros(5, 1)), "bias"),
    (dict(bias=torch.zeros(5).half()), "one dtype"),
    (dict(residual=torch.zeros(3, 4)), "residual"),
    (dict(residual=torch.zeros(5)), "residual"),
    (dict(residual=torch.zeros(3, 5).half()), "one dtype"),
    (dict(), "CUDA tensors only"),
    (dict(x=X.clone().requires_grad_()), "CUDA tensors only"),
])
def test_linear_refuses(kw, message):
    args = {"x": X, "weight": W, **kw}
    with pytest.raises(ValueError, match=message):
        attention.linear(**args)


Z, M = torch.zeros(3, 7), torch.ones(2, 7, dtype=torch.bool)
S, H = torch.zeros(3, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int64)


@pytest.mark.parametrize("kw,message", [
    (dict(logits=Z.double()), "float32, float16 or bfloat16"),
    (dict(logits=torch.zeros(())), "logits"),
    (dict(logits=torch.zeros(3, 0)), "operators"),
    (dict(logits=torch.zeros(1, 65537)), "operators"),
    (dict(tau=0.0), "positive"), (dict(tau=-1.0), "positive"), (dict(tau=float("nan")), "positive"),
    (dict(tau=float("inf")), "positive"), (dict(repetition=0.0), "positive"), (dict(repetition=float("nan")), "positive"),
    (dict(frequency=float("inf")), "finite"), (dict(presence=float("nan")), "finite"),
    (dict(bias=torch.zeros(6)), "bias"), (dict(bias=torch.zeros(7).half()), "bias"), (dict(bias=torch.zeros(1, 7)), "bias"),
    (dict(mask=torch.ones(2, 7)), "bool or uint8"),
    (dict(mask=M), "mask must be"),
    (dict(mask=M[:, :6], states=S), "mask must be"),
    (dict(mask=M[:0], states=S), "mask must be"),
    (dict(mask=M[0], states=S), "mask must be"),
    (dict(states=S), "next to a mask"),
    (dict(mask=M, states=S.int()), "states"),
    (dict(mask=M, states=S[:2]), "states"),
    (dict(history=H.int()), "history"), (dict(history=H[:2]), "history"), (dict(history=S[:2]), "history"),
    (dict(history=torch.zeros(3, 65536, dtype=torch.int64)), "65535"),
    (dict(mask=M, states=S, history=H, bias=torch.zeros(7)), "CUDA tensors only"),
])
def test_relation_weights_refuses(kw, message):
    with pytest.raises(ValueError, match=message):
        attention.relation_weights(**{"logits": Z, **kw})


P = torch.zeros(4, 6)


@pytest.mark.parametrize("kw,message", [
    (dict(update=P.double()), "float32, float16 or bfloat16"),
    (dict(update=torch.zeros(4)), "matrices"), (dict(update=torch.zeros(2, 0, 3)), "matrices"),
    (dict(steps=0), "steps"), (dict(steps=65), "steps"), (dict(steps=2.5), "steps"),
    (dict(coefficients=(1.0, 2.0)), "coefficients"), (dict(coefficients=(1.0, float("nan"), 0.0)), "coefficients"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(), "CUDA tensors only"),
])
def test_orthogonalize_refuses(kw, message):
    with pytest.raises(ValueError, match=message):
        muon.orthogonalize(**{"update": P, **kw})


@pytest.mark.parametrize("kw,message", [
    (dict(param=P.half()), "float32"), (dict(grad=torch.zeros(6, 4)), "float32"), (dict(momentum=P.double()), "float32"),
    (dict(lr=float("nan")), "lr"), (dict(beta=1.0), "beta"), (dict(beta=-0.1), "beta"),
    (dict(weight_decay=float("inf")), "weight_decay"), (dict(scale=float("inf")), "scale"),
    (dict(gate=torch.zeros(2)), "gate"), (dict(gate=torch.zeros(1).half()), "gate"),
    (dict(), "CUDA tensors only"),
])
def test_muon_update_refuses(kw, message):
    args = {"param": P.clone(), "grad": P.clone(), "momentum": P.clone(), "lr": 0.1, **kw}
    for f in (muon.muon_update, muon.muon_update_):
        with pytest.raises(ValueError, match=message):
            f(**args)


def test_in_place_update_refuses_overlapping_views():
    row = torch.zeros(1, 6).expand(4, 6)
    with pytest.raises(ValueError, match="overlap"):
        muon.muon_update_(row, P, P.clone(), lr=0.1)
    with pytest.raises(ValueError, match="overlap"):
        muon.muon_update_(P.clone(), P, torch.zeros(9).as_strided((4, 6), (1, 1)), lr=0.1)
    assert not muon._overlaps_itself(torch.zeros(3, 4, 5, 6).permute(1, 2, 0, 3))
    both = torch.zeros(2, 4, 6)
    for args in ((P, P, P.clone()), (P.clone(), P, P), (P, P.clone(), P), (both[0], both.view(-1)[20:44].view(4, 6), P)):
        with pytest.raises(ValueError, match="apart"):
            muon.muon_update_(*args, lr=0.1)
    with pytest.raises(ValueError, match="CUDA"):  # neighbours in one buffer are fine
        muon.muon_update_(both[0], both[1], P.clone(), lr=0.1)


def test_optimizer_refuses():
    with pytest.raises(ValueError, match="float32"):
        muon.Muon([torch.zeros(4, requires_grad=True)])
    with pytest.raises(ValueError, match="float32"):
        muon.Muon([torch.zeros(4, 4, dtype=torch.float16, requires_grad=True)])


def test_operator_rules_refuse():
    n, Q, T = 7, 3, 2
    ok = dict(mask=M, states=torch.zeros(T, Q, dtype=torch.int64), history=H, bias=torch.zeros(n))
    attention.OperatorRules(**ok).check(T, Q, n)
    for kw in (dict(states=None), dict(mask=None), dict(mask=M[:, :5]), dict(mask=M.float()), dict(states=S),
               dict(history=H[:2]), dict(history=H.int()), dict(bias=torch.zeros(6)), dict(bias=torch.zeros(n).half()),
               dict(repetition=0.0), dict(frequency=float("inf"))):
        with pytest.raises(ValueError):
            attention.OperatorRules(**{**ok, **kw}).check(T, Q, n)


@pytest.mark.parametrize("kw", [dict(optimizer="adam"), dict(table=torch.zeros(4, 3, 3, 6)),
                                dict(head=(torch.zeros(4, 6), None)), dict(head=(torch.zeros(5, 5), torch.zeros(4)))])
def test_step_refuses(kw):
    """Options that do not fit, refused before the graph is looked at."""
    with pytest.raises(ValueError):
        DrumTrainStep(None, 2, 4, 3, 3, None, 0, kw.pop("table", torch.zeros(4, 3, 3, 5)), n_hide=1, **kw)


# ---- the C ABI ------------------------------------------------------------------------------------
class Linear(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ("x", "w", "bias", "residual")] + \
               [(k, ctypes.c_int64) for k in ("ld_x", "ld_w", "ld_res", "rows", "n", "k")] + \
               [("dtype", ctypes.c_int), ("act", ctypes.c_int)]


class Weights(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ("logits", "bias", "mask", "states", "history")] + \
               [(k, ctypes.c_int64) for k in ("ld", "bias_ld", "mask_ld", "n_states", "hist_ld", "hist", "rows", "n")] + \
               [(k, ctypes.c_double) for k in ("tau", "repetition", "frequency", "presence")] + [("dtype", ctypes.c_int)]


def test_c_abi_refuses():
    """FL_EINVAL and a message, never an abort: bad sizes and types, missing arrays, small workspaces."""
    lib = L.lib()
    p = 0x1000  # never read: every call below is refused first
    good = dict(x=p, w=p, bias=None, residual=None, ld_x=4096, ld_w=4096, ld_res=0, rows=4096, n=4096, k=4096, dtype=0, act=0)
    for bad in (dict(dtype=7), dict(act=9), dict(n=0), dict(k=-1), dict(rows=-1), dict(x=None), dict(w=None), dict(ld_x=1),
                dict(residual=p, ld_res=3), dict(rows=1 << 40)):
        s = Linear(**{**good, **bad})
        assert lib.fl_linear_forward(ctypes.byref(s), p, 4096, None, p, 1 << 30, None) == 1
        assert lib.fl_linear_backward(ctypes.byref(s), None, p, 4096, p, p, p, p, 1 << 30, None) == 1
        assert lib.fl_last_error()
    s = Linear(**good)
    assert lib.fl_linear_forward(ctypes.byref(s), p, 4095, None, p, 1 << 30, None) == 1  # short output rows
    assert lib.fl_linear_forward(ctypes.byref(s), p, 4096, None, None, 0, None) == 1     # no workspace
    assert b"workspace" in lib.fl_last_error()
    assert lib.fl_linear_backward(ctypes.byref(Linear(**{**good, "act": 4})), None, p, 4096, p, p, p, p, 1 << 30, None) == 1
    for dims in ((0, 5, 5), (5, 0, 5), (5, 5, 0), (-3, 5, 5)):
        assert lib.fl_linear_workspace(*dims, 0) == 0 and lib.fl_linear_backward_workspace(*dims, 0, 3) == 0
    good = dict(logits=p, bias=None, mask=None, states=None, history=None, ld=100, rows=4, n=100, tau=1.0, repetition=1.0, dtype=0)
    for bad in (dict(n=0), dict(n=65537, ld=65537), dict(rows=-1), dict(ld=50), dict(logits=None), dict(tau=0.0),
                dict(repetition=-1.0), dict(dtype=3), dict(mask=p, n_states=0), dict(mask=p, n_states=2, mask_ld=50),
                dict(hist=5), dict(history=p, hist=70000)):
        w = Weights(**{**good, **bad})
        assert lib.fl_relation_weights(ctypes.byref(w), p, None) == 1
        assert lib.fl_relation_weights_backward(ctypes.byref(w), p, p, 100, p, None, p, 1 << 30, None) == 1
    assert lib.fl_relation_weights(ctypes.byref(Weights(**good)), None, None) == 1
    assert lib.fl_relation_weights_backward(ctypes.byref(Weights(**{**good, "bias": p})), p, p, 100, p, p, None, 0, None) == 1
    assert lib.fl_relation_weights_workspace(-1, 5) == 0 and lib.fl_relation_weights_workspace(5, 1 << 40) == 0

    class Matrices(ctypes.Structure):
        _fields_ = [("ptr", ctypes.c_void_p)] + [(k, ctypes.c_int64) for k in ("b1", "b2", "i", "j")]

    m = Matrices(p, 0, 0, 400, 1)
    r = ctypes.byref(m)
    c = (3.4445, -4.7750, 2.0315, 1e-7)
    for b1, b2, rows, cols, dtype, steps in ((1, 1, 0, 5, 0, 5), (1, 1, 5, 5, 4, 5), (1, 1, 5, 5, 0, 0), (1, 1, 5, 5, 0, 65),
                                             (-1, 1, 5, 5, 0, 5), (1, 1, 1 << 25, 5, 0, 5)):
        assert lib.fl_orthogonalize(r, r, b1, b2, rows, cols, dtype, steps, *c, p, 1 << 30, None) == 1
    assert lib.fl_orthogonalize(None, r, 1, 1, 400, 400, 0, 5, *c, p, 1 << 30, None) == 1
    assert lib.fl_orthogonalize(r, r, 1, 1, 400, 400, 0, 5, *c, None, 0, None) == 1
    assert lib.fl_orthogonalize(r, r, 1, 1, 400, 400, 0, 5, 30.0, 0.0, 0.0, 1e-7, p, 1 << 30, None) == 1  # runs away
    assert b"coefficients" in lib.fl_last_error()
    assert lib.fl_orthogonalize(None, None, 0, 1, 400, 400, 0, 5, *c, None, 0, None) == 0  # an empty batch
    assert lib.fl_muon_update(r, r, None, r, r, 1, 1, 400, 400, 0.1, 0.9, 1, 0.0, 1.0, 5, *c, None, p, 1 << 30, None) == 1
    assert lib.fl_newton_schulz_workspace(0, 5, 5, 5) == 0
