"""The exponential and the sigmoid that routing decides by, over their range, through the weights that they make.

e^x is 2^hi (off by 2^-22 at most: ex2.approx), times 1 + lo ln 2 (a rounding of the factor and one of the product, 2^-24 each):
below 1.5 2^-22.  A weight adds the rounding of a sum of two and of a quotient (2^-24 each; the sigmoid's quotient 2^-22): below
2^-21 for the softmax of two experts and 2^-20 for the sigmoid.  Values below the least normal number are zero."""
import pytest
import torch

from alto_b200 import routing

pytestmark = pytest.mark.gpu
TINY = 1.2e-38


def test_softmax_of_two():
    # 0 and -x: no rounding in front of the exponential
    x = torch.cat([torch.linspace(0, 90, 1 << 18), torch.linspace(0, 1, 1 << 16), 2.0 ** torch.linspace(-30, 0, 1 << 12)]).float()
    l = torch.stack([torch.zeros_like(x), -x], 1)
    ids, w = routing.route_experts(l.cuda(), 2, renormalize=False)
    want = torch.softmax(l.double(), -1).gather(1, ids.cpu().long())
    err = (w.cpu().double() - want).abs()
    assert (err <= want * 2.0 ** -21 + TINY).all(), float((err / want.clamp_min(TINY)).max() * 2 ** 21)


def test_sigmoid():
    l = torch.cat([torch.linspace(-95, 95, 1 << 18), torch.linspace(-1, 1, 1 << 16), -(2.0 ** torch.linspace(-30, 0, 1 << 12))]).float().unsqueeze(1)
    _, w = routing.route_experts(l.cuda(), 1, score="sigmoid", renormalize=False)
    want = torch.sigmoid(l.double())
    err = (w.cpu().double() - want).abs()
    assert (err <= want * 2.0 ** -20 + TINY).all(), float((err / want.clamp_min(TINY)).max() * 2 ** 20)
