"""Outputs of the norm and the routing may be written to, whatever the leading dimensions, as those of tensor operations may."""
import pytest
import torch

from alto_b200 import norm, routing

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64), (1, 2, 3, 64)])
def test_norm(shape):
    x = torch.randn(shape, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda")
    y = norm.rms_norm(x, w)
    y *= 2
    (g,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g, torch.autograd.grad(norm.rms_norm(x, w), x, torch.full(shape, 2.0, device="cuda"))[0])
    y, r = norm.rms_norm(x, w, residual=x)
    y += 1
    r.detach()
    torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64), (1, 2, 3, 64)])
def test_routing(shape):
    logits = torch.randn(shape, device="cuda", requires_grad=True)
    ids, weights = routing.route_experts(logits, 4)
    weights *= 3
    (g,) = torch.autograd.grad(weights, logits, torch.arange(weights.numel(), device="cuda").view(weights.shape).float())
    _, again = routing.route_experts(logits, 4, scale=3.0)
    want = torch.autograd.grad(again, logits, torch.arange(weights.numel(), device="cuda").view(weights.shape).float())[0]
    # either gradient q (g - sum g q) 3 is off by at most 4 2^-18 of q (|g| + sum |g| q) 3, whose factor of q is at most 6 numel
    atol = 2 * 4 * 2.0 ** -18 * 6 * weights.numel()
    assert ids.shape == weights.shape == shape[:-1] + (4,) and ((g - want).abs() <= atol).all()
