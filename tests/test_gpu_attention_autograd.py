"""What autograd is told about the relation attention: a second derivative is an error whichever input it is of, and so
are forward-mode derivatives."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def head(dt=torch.float32, rows=20, k=12, n=10):
    g = torch.Generator().manual_seed(3)
    return ((torch.randn(rows, k, generator=g)).to(dt).cuda(), (torch.randn(n, k, generator=g)).to(dt).cuda(),
            torch.randn(n, generator=g).to(dt).cuda())


def assert_second_is_an_error(y, leaf):
    grad, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    assert grad.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        grad.square().sum().backward()


@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
@pytest.mark.parametrize("which", [0, 1, 2], ids=["x", "weight", "bias"])
def test_second_derivative_of_the_only_leaf(which, act):
    """With an activation every gradient depends on every input, through the pre-activation."""
    from flashlog_b200 import attention
    ts = list(head())
    ts[which] = ts[which].requires_grad_()
    assert_second_is_an_error(attention.linear(*ts, activation=act), ts[which])


@pytest.mark.parametrize("of", [0, 1], ids=["x", "weight"])
def test_second_derivative_through_the_other_operand(of):
    """Without one, dx depends on the weight and dweight on x."""
    from flashlog_b200 import attention
    x, w, _ = head()
    x.requires_grad_(), w.requires_grad_()
    assert_second_is_an_error(attention.linear(x, w), (x, w)[of])


@pytest.mark.parametrize("which", [0, 1], ids=["logits", "bias"])
@pytest.mark.parametrize("wide", [False, True])
def test_second_derivative_of_weights(which, wide):
    from flashlog_b200 import attention
    g = torch.Generator().manual_seed(5)
    z = torch.randn(6, 40, generator=g).cuda()
    b = torch.randn(*((6, 40) if wide else (40,)), generator=g).cuda()
    (z, b)[which].requires_grad_()
    coefficients = torch.randn(6, 40, generator=g).cuda()
    assert_second_is_an_error(attention.relation_weights(z, bias=b) * coefficients, (z, b)[which])


def test_gradients_that_depend_on_nothing_need_no_graph():
    """dx of a linear map whose weight is a constant is a constant: a penalty on it has no second derivative."""
    from flashlog_b200 import attention
    x, w, b = head()
    x.requires_grad_(), b.requires_grad_()
    gx, gb = torch.autograd.grad(attention.linear(x, w, b).sum(), (x, b), create_graph=True)
    assert not gx.requires_grad and not gb.requires_grad


@pytest.mark.parametrize("which", range(4), ids=["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_of_linear_is_an_error(which, leaf):
    """Also for tensors that require no gradient."""
    import torch.autograd.forward_ad as fwd
    from flashlog_b200 import attention
    ts = [*head(), torch.ones(20, 10).cuda()]
    if leaf:
        ts[0].requires_grad_()
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ts[which] = fwd.make_dual(ts[which], torch.ones_like(ts[which]))
        attention.linear(*ts)


@pytest.mark.parametrize("which", [0, 1], ids=["logits", "bias"])
def test_forward_mode_of_weights_is_an_error(which):
    import torch.autograd.forward_ad as fwd
    from flashlog_b200 import attention
    ts = [torch.ones(6, 40).cuda(), torch.ones(40).cuda()]
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ts[which] = fwd.make_dual(ts[which], torch.ones_like(ts[which]))
        attention.relation_weights(ts[0], bias=ts[1])


def test_forward_mode_of_updates_is_an_error():
    import torch.autograd.forward_ad as fwd
    from flashlog_b200 import muon
    u = torch.randn(6, 40).cuda()
    with fwd.dual_level():
        dual = fwd.make_dual(u, torch.ones_like(u))
        with pytest.raises(RuntimeError, match="forward-mode"):
            muon.orthogonalize(dual)
        with pytest.raises(RuntimeError, match="forward-mode"):
            muon.muon_update(u, dual, torch.zeros_like(u), lr=0.1)
