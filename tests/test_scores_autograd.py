"""The differentiable functions of the score operators as autograd sees them.  No GPU: plain torch
forms stand in for the kernels."""
import pytest
import torch

from filtervectorcode_refactor_amd import scores as S


@pytest.fixture
def plain(monkeypatch):
    def quantize_fp8(x, block="row", transpose=False):
        return (x, None, x.t(), None) if transpose else (x, None)

    def distill_forward(scores, ids, values, teacher_lse=None, temperature=1.0):
        return torch.logsumexp(scores, dim=1), scores

    monkeypatch.setattr(S, "quantize_fp8", quantize_fp8)
    monkeypatch.setattr(S, "_transposed", lambda x: (x.t(), None))
    monkeypatch.setattr(S, "matmul_fp8", lambda a, _, b, __, dtype=None: a @ b.t())
    monkeypatch.setattr(S, "matmul_fp8_grad", lambda g, xt, _, wt, __: (g @ wt.t(), g.t() @ xt.t()))
    monkeypatch.setattr(S, "distill_forward", distill_forward)
    monkeypatch.setattr(S, "distill_backward",
                        lambda w, s, ids, values, saved, teacher_lse=None, temperature=1.0: w[:, None] * s.softmax(1))


def _twice(y, of):
    """Both passes of a loss of the result and of its gradient's square."""
    (first,) = torch.autograd.grad(y.sum(), of, create_graph=True)
    (y.sum() + first.square().sum()).backward()


@pytest.mark.parametrize("of", ["x", "w"])
def test_linear_has_no_second_derivative(plain, of):
    """Its gradient is made by kernels that autograd does not see: a gradient of it is refused, not
    taken as 0."""
    t = {"x": torch.randn(5, 8), "w": torch.randn(6, 8)}
    t[of].requires_grad_()
    y = S._LinearFp8.apply(t["x"], t["w"], torch.float32)
    with pytest.raises(RuntimeError, match="no second derivative"):
        _twice(y.square(), t[of])


def test_linear_gradients_depend_on_the_other_operand(plain):
    """dx = g w with a constant g: the derivative by w is refused too."""
    x, w = torch.randn(5, 8, requires_grad=True), torch.randn(6, 8, requires_grad=True)
    (dx,) = torch.autograd.grad(S._LinearFp8.apply(x, w, torch.float32).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        dx.square().sum().backward()
    assert w.grad is None


def test_distill_loss_has_no_second_derivative(plain):
    s = torch.randn(5, 8, requires_grad=True)
    loss = S.distill_loss(s, torch.zeros(5, 1), torch.zeros(5, 1))
    with pytest.raises(RuntimeError, match="no second derivative"):
        _twice(loss, s)


@pytest.mark.parametrize("create_graph", [False, True])
def test_first_derivatives(plain, create_graph):
    x, w = torch.randn(5, 8, requires_grad=True), torch.randn(6, 8, requires_grad=True)
    up = torch.randn(5, 6)
    dx, dw = torch.autograd.grad(S._LinearFp8.apply(x, w, torch.float32), (x, w), up, create_graph=create_graph)
    assert torch.equal(dx, up @ w.detach()) and torch.equal(dw, up.t() @ x.detach())
    assert dx.requires_grad == dw.requires_grad == create_graph
    for t in (x, w):
        y = S._LinearFp8.apply(*(a if a is t else a.detach() for a in (x, w)), torch.float32)
        (got,) = torch.autograd.grad(y, t, up, create_graph=create_graph)
        assert torch.equal(got, dx if t is x else dw)
    s = torch.randn(5, 8, requires_grad=True)
    loss = S.distill_loss(s, torch.zeros(5, 1), torch.zeros(5, 1)).sum()
    assert torch.equal(torch.autograd.grad(loss, s, create_graph=create_graph)[0], s.detach().softmax(1))
