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


def saved_by_a_graph(shape, strided):
    """A leaf (a contiguous one, or a view of a wider table) and the loss of a graph that saved it."""
    base = torch.randn(shape[0], 2, shape[1]).cuda()
    w = base.permute(1, 0, 2) if strided else base.permute(1, 0, 2).contiguous()
    w.requires_grad_()
    return w, w.square().sum()


@pytest.mark.parametrize("shape", [(20, 30), (300, 280)], ids=str)  # one block; the tensor path
@pytest.mark.parametrize("strided", [False, True])
def test_updates_in_place_are_seen_by_autograd(shape, strided):
    """As after torch's own optimizers: a graph that saved the parameter before the step cannot run on the new one."""
    from flashlog_b200 import muon
    w, loss = saved_by_a_graph(shape, strided)
    w.grad = torch.randn_like(w)
    before = w._version
    optimizer = muon.Muon([w], lr=0.1)
    optimizer.step()
    momentum = optimizer.state[w]["momentum"]
    assert w._version > before and momentum._version > 0
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


def test_outputs_given_by_the_caller_are_seen_by_autograd():
    from flashlog_b200 import ops
    x, w, b = head()
    out = torch.empty(20, 10).cuda().requires_grad_()
    loss = out.square().sum()
    with torch.no_grad():
        ops.linear_forward(x, w, b, out=out)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    out = torch.empty(20, 10).cuda().requires_grad_()
    loss = out.square().sum()
    with torch.no_grad():
        ops.relation_weights(x @ w.T, out=out)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


def test_updates_of_inference_tensors_run():
    from flashlog_b200 import muon
    with torch.inference_mode():
        p, g, m = (torch.randn(20, 30).cuda() for _ in range(3))
        q, n = muon.muon_update(p, g, m, lr=0.1)
        muon.muon_update_(p, g, m, lr=0.1)
    assert torch.equal(p, q) and torch.equal(m, n)
    muon.muon_update_(p, g, m, lr=0.1)
