"""Forward-mode differentiation is refused by every operator that has a gradient, not passed by without one."""
import pytest
import torch
from torch.autograd import forward_ad

from alto_b200 import norm, routing
from alto_b200.swiglu import swiglu

pytestmark = pytest.mark.gpu


def _calls(dual):
    x, t = torch.randn(32, 128, device="cuda").bfloat16(), torch.randn(32, 128, device="cuda").bfloat16()
    w, wt = torch.ones(128, device="cuda").bfloat16(), torch.randn(128, device="cuda").bfloat16()
    return [lambda: norm.rms_norm(dual(x, t), w), lambda: norm.rms_norm(x, dual(w, wt)), lambda: norm.rms_norm(x, w, residual=dual(x, t)),
            lambda: norm.rms_norm_mxfp8_linear(dual(x, t), w, x), lambda: routing.route_experts(dual(x, t), 4),
            lambda: swiglu(dual(x, t)), lambda: swiglu(dual(x, t), checkpoint="e4m3")]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", range(7))
def test_a_tangent_is_not_dropped(which, grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError):
            _calls(forward_ad.make_dual)[which]()


def test_tensors_without_a_tangent_are_taken_at_a_dual_level():
    x, w = torch.randn(32, 128, device="cuda").bfloat16(), torch.ones(128, device="cuda").bfloat16()
    want = (norm.rms_norm(x, w), *norm.rms_norm(x, w, residual=x), *routing.route_experts(x, 4))
    with forward_ad.dual_level():
        got = (norm.rms_norm(x, w), *norm.rms_norm(x, w, residual=x), *routing.route_experts(x, 4))
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))
