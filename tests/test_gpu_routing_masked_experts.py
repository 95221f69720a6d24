"""Experts masked by their bias: -inf, the type's lowest value, or a large negative number, with groups judged by their two
best keys.  No tolerance: the chosen experts are those of the definition in 64 bits."""
import pytest
import torch

from alto_b200 import routing

pytestmark = pytest.mark.gpu


def _choice64(logits, k, score, bias, groups, kept, top):
    s = torch.sigmoid(logits.double()) if score == "sigmoid" else torch.softmax(logits.double(), -1)
    key = s + bias.double()
    of = torch.sort(key.unflatten(-1, (groups, -1)), dim=-1, descending=True).values[..., :top].sum(-1)
    order = torch.sort(of, dim=-1, descending=True, stable=True).indices
    out = torch.ones_like(of, dtype=torch.bool).scatter(-1, order[..., :kept], False).repeat_interleave(key.shape[-1] // groups, -1)
    first = torch.sort(key, dim=-1, descending=True, stable=True).indices      # dropped experts behind kept ones of -inf
    return first.gather(-1, torch.sort(out.gather(-1, first).int(), dim=-1, stable=True).indices)[..., :k]


# groups inside a lane, of whole lanes, and neither (the form through shared memory)
SHAPES = [(256, 32), (64, 32), (512, 32), (256, 8), (48, 16), (96, 3), (120, 8), (32, 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("mask", [-torch.inf, torch.finfo(torch.float32).min, -1e9])
@pytest.mark.parametrize("experts, groups", SHAPES)
def test_masked_groups_and_groups_with_one_expert_left(experts, groups, mask, score, dtype):
    g = torch.Generator().manual_seed(experts + groups)
    size = experts // groups
    l = torch.randn(300, experts, generator=g).to(dtype)
    plain = torch.randn(experts, generator=g) * 0.1
    whole, single, last = plain.clone(), plain.clone(), plain.clone()
    whole[:size] = mask                                        # the first group, whole
    whole[size * (groups - 1):] = mask                         # and the last
    single[:size] = mask
    single[size - 1] = 0.3                                     # the last expert of the first group is left
    single[size:2 * size] = mask
    single[size] = 0.2                                         # the first expert of the second
    last[:] = mask                                             # one group is left, which is not the first
    last[size * (groups - 1):] = plain[size * (groups - 1):]
    for bias in (whole, single, last):
        for kept in {1, 2, groups - 1}:
            for top in (1, 2):
                for k in {1, min(16, kept * size)}:
                    ids, weights = routing.route_experts(l.cuda(), k, score=score, bias=bias.cuda(), num_groups=groups, groups_kept=kept,
                                                         group_top=top)
                    want = _choice64(l, k, score, bias, groups, kept, top)
                    assert torch.equal(ids.cpu().long(), want), (kept, top, k)
                    assert torch.isfinite(weights).all()


@pytest.mark.parametrize("experts, groups", SHAPES)
def test_experts_that_are_always_taken(experts, groups):
    # a bias of +inf: its group comes first, and among several such groups the lowest
    g = torch.Generator().manual_seed(experts)
    size = experts // groups
    l = torch.randn(200, experts, generator=g)
    bias = torch.randn(experts, generator=g) * 0.1
    for at in ((experts - 1,), (experts - 1, size), (size, 2 * size + size - 1)):
        taken = bias.clone()
        taken[list(at)] = torch.inf
        for kept in (1, 2):
            for top in (1, 2):
                ids, _ = routing.route_experts(l.cuda(), 1, score="sigmoid", bias=taken.cuda(), num_groups=groups, groups_kept=kept, group_top=top)
                assert torch.equal(ids.cpu().long(), _choice64(l, 1, "sigmoid", taken, groups, kept, top))
