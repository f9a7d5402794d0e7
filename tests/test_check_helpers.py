"""The helpers that operators share, on the CPU: backwards that cannot be differentiated, saved tensors as kernels read them."""
import pytest
import torch

from eacs_b200.ops._check import once, packed


class Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, power):
        ctx.save_for_backward(x, w)
        return x * w

    @staticmethod
    @once
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        return dy * w, dy * x if ctx.needs_input_grad[1] else None, None


def test_once_gives_gradients_that_raise_when_they_are_differentiated():
    x, w = torch.randn(5, requires_grad=True), torch.randn(5, requires_grad=True)
    plain = torch.autograd.grad(Product.apply(x, w, 1).sum(), (x, w))
    assert not plain[0].requires_grad and torch.equal(plain[0], w) and torch.equal(plain[1], x)
    for upstream in (torch.ones(5), torch.ones(5, requires_grad=True)):
        made = torch.autograd.grad(Product.apply(x, w, 1), (x, w), upstream, create_graph=True)
        assert torch.equal(made[0], w) and torch.equal(made[1], x)
        for g in made:
            with pytest.raises(RuntimeError, match="differentiated once"):
                torch.autograd.grad(g.sum(), x, allow_unused=True, retain_graph=True)
            with pytest.raises(RuntimeError, match="differentiated once"):  # a penalty among terms that do have a gradient
                torch.autograd.grad(g.square().sum() + x.square().sum(), x, retain_graph=True)
    only = torch.autograd.grad(Product.apply(x, w.detach(), 1).sum(), x, create_graph=True)[0]  # (an input that wants none)
    assert torch.equal(only, w)
    y = Product.apply(x, w, 1).sum()
    for _ in range(2):
        assert torch.equal(torch.autograd.grad(y, x, retain_graph=True)[0], w)


def test_packed():
    assert packed(None) is None
    t = torch.arange(12.0).view(3, 4)
    assert packed(t) is t or packed(t).data_ptr() == t.data_ptr()
    apart = torch.empty(3, 4, 2)[..., 0].copy_(t)
    shifted = torch.empty(13)[1:].view(3, 4).copy_(t)
    for odd in (apart, shifted, t.t().contiguous().t()):
        p = packed(odd)
        assert torch.equal(p, t) and p.is_contiguous() and p.data_ptr() % 16 == 0
