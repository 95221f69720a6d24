"""A group masked by a large negative bias takes part in no close decision, so the tokens keep the fp32 path."""
import pytest
import torch

from alto_b200 import routing

pytestmark = pytest.mark.gpu


def _time(call):
    for _ in range(3):
        call()
    best = float("inf")
    for _ in range(5):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(4):
            call()
        end.record()
        end.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


@pytest.mark.parametrize("experts, groups", [(256, 8), (96, 3)])
@pytest.mark.parametrize("mask", [-1e4, -1e9, torch.finfo(torch.float32).min, -torch.inf])
def test_a_masked_group_does_not_make_every_token_uncertain(mask, experts, groups):
    # a token done again in double takes ten times its time and more; close decisions make up a fraction of a percent
    l = torch.randn(65536, experts, generator=torch.Generator().manual_seed(0)).cuda()
    bias = torch.zeros(experts, device="cuda")
    masked = bias.clone()
    masked[:experts // groups] = mask
    took = [_time(lambda: routing.route_experts(l, 4, score="sigmoid", bias=b, num_groups=groups, groups_kept=2, group_top=2)) for b in (bias, masked)]
    assert took[1] <= 2.0 * took[0], took
