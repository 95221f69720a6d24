"""Choices between keys a few steps of fp32 apart, from lanes that hold many experts: a key is compared without the bits that
say which of its lane's experts it is, so those bits take part in no decision.

No tolerance: the chosen experts are those of the definition in 64 bits."""
import math

import pytest
import torch

from alto_b200 import routing

pytestmark = pytest.mark.gpu
ROWS = 1 << 16


# 64, 256 and 512 experts: 2, 8 and 16 a lane; the first expert of one lane and the last of another, in either order
@pytest.mark.parametrize("experts, per", [(64, 2), (256, 8), (512, 16), (250, 8)])
@pytest.mark.parametrize("target", [0.5, 1.0, 1.5, 2.0])
@pytest.mark.parametrize("low, high", [(0.1, 0.13), (0.3, 0.5), (0.05, 0.6), (0.6, 0.9)])
def test_first_and_last_expert_of_two_lanes(low, high, target, experts, per):
    g = torch.Generator(device="cuda").manual_seed(experts)
    step = 2.0 ** -23 * (target if target >= 1 else 0.5)
    for a, b in ((3 * per, 20 * per + per - 1), (3 * per + per - 1, 20 * per)):
        # different scores under biases that bring both keys to `target`, then two steps of fp32 apart at most
        bias = torch.full((experts,), -5.0, device="cuda")
        bias[a], bias[b] = target - low, target - high
        l = torch.randn(ROWS, experts, generator=g, device="cuda") * 0.1 - 6.0
        l[:, a] = math.log(low / (1 - low)) + torch.randn(ROWS, generator=g, device="cuda") * 2e-3
        apart = (torch.rand(ROWS, generator=g, device="cuda").double() * 4 - 2) * step
        l[:, b] = torch.logit(torch.sigmoid(l[:, a].double()) + bias[a].double() + apart - bias[b].double()).float()
        key = torch.sigmoid(l[:, [a, b]].double()) + bias[[a, b]].double()
        assert ((key[:, 0] - key[:, 1]).abs() < 2 * step).float().mean() > 0.95     # the case is what it says it is
        want = torch.where(key[:, 1] > key[:, 0], b, a)
        for k in (1, 2):      # the last choice against its successor, and two choices against one another
            ids, _ = routing.route_experts(l, k, score="sigmoid", bias=bias)
            assert torch.equal(ids[:, 0].long(), want), (k, int((ids[:, 0] != want).sum()))


@pytest.mark.parametrize("experts", [256, 512])
def test_many_near_keys(experts):
    # all experts' keys within some steps of one another in every row
    g = torch.Generator().manual_seed(experts)
    base = torch.randn(experts, generator=g)
    l = (base.view(torch.int32) + torch.randint(-4, 5, (2000, experts), generator=g).int()).view(torch.float32)
    bias = (0.75 - torch.sigmoid(base.double())).float()
    order = torch.sort(torch.sigmoid(l.double()) + bias.double(), dim=-1, descending=True, stable=True).indices
    for k in (1, 8, 16):
        ids, _ = routing.route_experts(l.cuda(), k, score="sigmoid", bias=bias.cuda())
        assert torch.equal(ids.cpu().long(), order[:, :k])


def test_scores_below_the_least_normal_number():
    # a score that fp32 flushes to zero beside a bias of its own size
    l = torch.full((400, 64), -200.0)
    bias = torch.zeros(64)
    l[:, 9] = -90.0 + torch.rand(400, generator=torch.Generator().manual_seed(0)) * 4      # scores of 8e-40 to 4.5e-38
    bias[9], bias[40] = 1.2e-38, 1.4e-38
    key = torch.sigmoid(l.double()) + bias.double()
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    assert set(order[:, 0].tolist()) == {9, 40}
    for k in (1, 2):
        ids, _ = routing.route_experts(l.cuda(), k, score="sigmoid", bias=bias.cuda())
        assert torch.equal(ids.cpu().long(), order[:, :k])
    for top in (1, 2):
        ids, _ = routing.route_experts(l.cuda(), 1, score="sigmoid", bias=bias.cuda(), num_groups=8, groups_kept=1, group_top=top)
        assert torch.equal(ids.cpu().long(), order[:, :1])
