"""NaN logits of a softmax: every score of the token is NaN, whichever experts are chosen."""
import pytest
import torch

from alto_b200 import routing

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("options", [dict(), dict(num_groups=4, groups_kept=2, group_top=1), dict(num_groups=4, groups_kept=2, group_top=2),
                                     dict(num_groups=4, groups_kept=4, group_top=2), dict(num_groups=16, groups_kept=2, group_top=2)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_a_token_with_a_nan_has_no_other_weights(with_bias, options, renormalize, dtype):
    clean = torch.randn(12, 64, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    logits = clean.clone()
    logits[2, 0] = logits[5, 33] = logits[9, 63] = torch.nan
    bias = torch.zeros(64, device="cuda") if with_bias else None
    ids, weights = routing.route_experts(logits, 6, bias=bias, renormalize=renormalize, **options)
    assert ids.min() >= 0 and ids.max() < 64 and (ids.sort(-1).values.diff(dim=-1) > 0).all()
    assert torch.isnan(weights[[2, 5, 9]]).all()
    rest = [i for i in range(12) if i not in (2, 5, 9)]
    want = routing.route_experts(clean, 6, bias=bias, renormalize=renormalize, **options)
    assert torch.equal(ids[rest], want[0][rest]) and torch.equal(weights[rest], want[1][rest])
