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


@pytest.mark.parametrize("shape", [(64, 128), (2, 32, 128)])
@pytest.mark.parametrize("residual", [False, True])
def test_linears_behind_a_norm(shape, residual):
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(shape, generator=g, device="cuda").bfloat16().requires_grad_(True)
    w, nw = torch.randn(96, 128, generator=g, device="cuda").bfloat16().requires_grad_(True), torch.ones(128, device="cuda").bfloat16()
    res = x.detach().clone().requires_grad_(True) if residual else None
    up = torch.randn(*shape[:-1], 96, generator=g, device="cuda").bfloat16()
    results = []
    for in_place in (True, False):
        got = norm.rms_norm_mxfp8_linear(x, nw, [w, w], residual=res)
        assert len(got) == (3 if residual else 2) and all(t.shape[:-1] == x.shape[:-1] for t in got)
        q = got[0].mul_(2) if in_place else got[0] * 2
        loss = (q * up).sum() + (got[1] * up).sum() + (got[2].sum() if residual else 0)
        results.append(torch.autograd.grad(loss, (x, w, res) if residual else (x, w)))
    assert all(torch.equal(a, b) for a, b in zip(*results)) and results[0][0].shape == x.shape
