"""The dispatcher's two ways on one rank agree, bit for bit, on slots without an expert."""
import pytest
import torch

from alto_b200 import _lib as L
from alto_b200 import distributed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("empty", [False, True])
def test_both_ways(dtype, empty, monkeypatch):
    g = torch.Generator().manual_seed(0)
    x, dy = torch.randn(300, 64, generator=g).cuda().to(dtype), torch.randn(300, 64, generator=g).cuda().to(dtype)
    ids = torch.full((300, 3), 8) if empty else torch.randint(-3, 12, (300, 3), generator=g)
    scores = torch.rand(300, 3, generator=g).cuda()
    got = []
    for general in (False, True):
        if general:
            monkeypatch.setattr(L, "on_current_device", lambda t: False)
        leaf, w = x.clone().requires_grad_(True), scores.clone().requires_grad_(True)
        d = distributed.ExpertParallelDispatcher(8)
        local, offs, state = d.dispatch(leaf, ids.cuda())
        out = d.combine(local * 2, state, w)
        got.append((local.detach(), offs, out.detach(), *torch.autograd.grad(out, (leaf, w), dy), d.combine(local.detach(), state)))
    for a, b in zip(*got):
        assert a.dtype == b.dtype and torch.equal(a, b)
    assert not empty or (got[0][2] == 0).all()
