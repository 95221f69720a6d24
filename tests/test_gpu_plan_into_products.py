"""The row plan straight into the grouped products: a buffer of the default size, longer than the runs, and one that the plan
does not fit into, whose last runs are cut off."""
import pytest
import torch

from alto_b200 import _lib as L
from alto_b200 import grouped, routing

pytestmark = pytest.mark.gpu

PRODUCTS = {
    "mxfp8": lambda a, w, offs: grouped._quantize_then_mxfp8_scaled_grouped_mm(a, w, offs),
    "mxfp4": lambda a, w, offs: grouped._quantize_then_mxfp_scaled_grouped_mm(a, w, offs, False, True, False, False, False, "none", False),
    "mxfp4 two-level": lambda a, w, offs: grouped._quantize_then_mxfp_scaled_grouped_mm(a, w, offs, False, True, False, False, False, "none", True),
    "nvfp4": lambda a, w, offs: grouped._quantize_then_nvfp4_scaled_grouped_mm(a, w, offs, False, True, False, use_outer_scale=True),
}


def _inputs(tokens, k, experts, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, 256, generator=g, device="cuda").bfloat16()
    w = (torch.randn(experts, 128, 256, generator=g, device="cuda") * 0.05).bfloat16()
    ids, _ = routing.route_experts(torch.randn(tokens, experts, generator=g, device="cuda"), k)
    return x, w, ids


def _step(product, rows, w, offs, dy):
    leaf, wl = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = PRODUCTS[product](leaf, wl.transpose(-2, -1), offs)
    return y.detach(), *torch.autograd.grad(y, (leaf, wl), dy)


@pytest.mark.parametrize("product", PRODUCTS)
def test_default_rows_without_a_look_at_the_counts(product):
    x, w, ids = _inputs(700, 2, 8, 0)
    plan = routing.expert_plan(ids, 8)
    rows, end = plan.token.numel(), int(plan.offs[-1])
    assert end < rows
    buffer = L.gather_rows(x, plan.token)
    dy = torch.randn(rows, 128, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").bfloat16()
    dy = torch.where((plan.token < 0).unsqueeze(1), torch.zeros_like(dy), dy)      # as combine's gradient gives it
    whole, cut = _step(product, buffer, w, plan.offs, dy), _step(product, buffer[:end], w, plan.offs, dy[:end])
    for a, b in zip(whole[:2], cut[:2]):
        assert torch.equal(a[:end], b) and (a[end:] == 0).all()
    assert torch.equal(whole[2], cut[2])


@pytest.mark.parametrize("product", PRODUCTS)
@pytest.mark.parametrize("rows", [128, 640, 1024, 1056, 160])
def test_a_buffer_that_is_too_short(product, rows):
    x, w, ids = _inputs(700, 2, 8, 1)
    plan = routing.expert_plan(ids, 8, rows=rows)
    assert int(plan.offs[-1]) > rows
    buffer = L.gather_rows(x, plan.token)
    dy = torch.randn(rows, 128, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").bfloat16()
    got, want = _step(product, buffer, w, plan.offs, dy), _step(product, buffer, w, plan.offs.clamp(max=rows), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    beyond = (torch.cat([plan.offs.new_zeros(1), plan.offs[:-1]]) >= rows).nonzero().flatten()
    assert len(beyond) > 0 and (got[2][beyond] == 0).all() and torch.isfinite(got[2]).all()
