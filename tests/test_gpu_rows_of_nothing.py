"""Row gather, combine and spread from buffers without a row: what a rank that received nothing hands over."""
import pytest
import torch

from alto_b200 import _lib as L
from alto_b200 import distributed

pytestmark = pytest.mark.gpu


def test_sources_without_rows_give_zeros():
    none = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    index = torch.tensor([-1, 0, 5, -1, 2, 7], dtype=torch.int32, device="cuda")
    out = L.gather_rows(none, index)
    assert out.shape == (6, 64) and (out == 0).all()
    out = L.combine_rows(none, index, torch.ones(3, 2, device="cuda").bfloat16(), 3, 2)
    assert out.shape == (3, 64) and (out == 0).all()
    out = L.spread_rows(none, index, None, 2)
    assert out.shape == (6, 64) and (out == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dispatch_without_tokens(dtype):
    x = torch.empty(0, 64, device="cuda", dtype=dtype, requires_grad=True)
    d = distributed.ExpertParallelDispatcher(4)
    local, offs, state = d.dispatch(x, torch.empty(0, 2, device="cuda", dtype=torch.int64))
    assert local.shape == (512, 64) and (local == 0).all() and offs.tolist() == [128, 256, 384, 512]
    out = d.combine(local, state, torch.empty(0, 2, device="cuda"))
    assert out.shape == (0, 64)
    out.sum().backward()
    assert x.grad.shape == (0, 64)
