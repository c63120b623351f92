"""gated.first_derivatives_only on a Function of its own: first derivatives under create_graph=True, no second ones."""
import pytest
import torch

from flashmlp_amd.gated import first_derivatives_only


class Square(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, n):
        ctx.save_for_backward(x)
        return x * x

    @staticmethod
    @first_derivatives_only
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        return 2 * x * g, None


@pytest.mark.parametrize("constant", [True, False])
def test_once(constant):
    x = torch.arange(4.0, requires_grad=True)
    y = Square.apply(x, 3)
    loss = y.sum() if constant else y.square().sum()  # (an incoming gradient that is a constant, or depends on x)
    (plain,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert not plain.requires_grad
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    assert torch.equal(g, plain) and g.requires_grad
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(g.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        (loss + g.square().sum()).backward()
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(Square.apply(x, 1).sum() + g.square().sum(), x)
