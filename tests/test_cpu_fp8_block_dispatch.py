"""The schemes fp8_block_e4m3 and fp8_block_e5m2: routing of wrapped weights, what they refuse, the modifier.  No kernel is launched."""
import pytest
import torch
from torch import nn

import alto_b200.dispatch as D
from alto_b200.dispatch import FP8BlockTrainingWeightWrapperTensor as Wrapped
from alto_b200.dispatch import TrainingOpConfig, swap_params
from alto_b200.lpt import LowPrecisionTrainingModifier


def config(**kw):
    base = dict(precision="fp8_block_e4m3", use_2dblock_x=False, use_2dblock_w=True, use_hadamard=False, use_sr_grad=False, use_dge=False)
    base.update(kw)
    return TrainingOpConfig(**base)


@pytest.fixture
def calls(monkeypatch):
    got = []

    def linear(a, b, **kw):
        got.append((a, b, kw))
        return torch.zeros(*a.shape[:-1], b.shape[0])

    def grouped(a, b, **kw):
        got.append((a, b, kw))
        return torch.zeros(a.shape[0], b.shape[-1])
    monkeypatch.setattr(D, "_to_fp8_block_then_scaled_mm", linear)
    monkeypatch.setattr(D, "_quantize_then_fp8_block_scaled_grouped_mm", grouped)
    return got


@pytest.mark.parametrize("variant", ["e4m3", "e5m2"])
def test_linear_and_products(calls, variant):
    w, x = Wrapped(torch.randn(16, 32), config(precision=f"fp8_block_{variant}")), torch.randn(4, 32)
    y = nn.functional.linear(x, w, torch.ones(16))
    assert torch.equal(y, torch.ones(4, 16))
    torch.matmul(x, w.t())
    torch.ops.aten.mm.default(x, w.t())
    assert [c[1].shape for c in calls] == [(16, 32)] * 3 and all(torch.equal(c[0], x) for c in calls)
    assert isinstance(calls[0][1], Wrapped)
    assert all(c[2] == dict(fp8_variant=variant) for c in calls)


def test_grouped(calls):
    w, x, offs = Wrapped(torch.randn(2, 16, 32), config()), torch.randn(6, 32), torch.tensor([2, 6], dtype=torch.int32)
    assert torch._grouped_mm(x, w.transpose(-2, -1), offs=offs).shape == (6, 16)
    assert calls[0][1].shape == (2, 32, 16) and calls[0][2]["offs"] is offs and calls[0][2]["fp8_variant"] == "e4m3"


@pytest.mark.parametrize("change", [dict(use_2dblock_w=False), dict(use_2dblock_x=True), dict(use_hadamard=True), dict(use_sr_grad=True),
                                    dict(use_dge=True), dict(use_uos=True), dict(clip_mode="static"), dict(two_level_scaling="tensorwise"),
                                    dict(precision="mxfp8_e4m3")], ids=str)
def test_options_it_has_not(calls, change):
    w = Wrapped(torch.randn(16, 32), config(**change))
    with pytest.raises(AssertionError):
        nn.functional.linear(torch.randn(4, 32), w)
    with pytest.raises(AssertionError):
        torch._grouped_mm(torch.randn(4, 32), Wrapped(torch.randn(1, 32, 16), config(**change)), offs=torch.tensor([4], dtype=torch.int32))
    assert not calls


def test_wrapping():
    p = swap_params(nn.Parameter(torch.randn(16, 16)), config=config(precision="fp8_block_e5m2"))
    assert isinstance(p.data, Wrapped) and isinstance(p.detach(), Wrapped) and isinstance(p.data.to(torch.bfloat16), Wrapped)
    assert D.quantized_gather_plan(torch.randn(128, 128), config(), None) is None       # its shards travel as they are
    (p * 2.0).sum().backward()
    assert p.grad.shape == (16, 16)


def test_modifier():
    class GroupedExperts(nn.Module):
        def __init__(self):
            super().__init__()
            self.w1 = nn.Parameter(torch.randn(2, 16, 32))

    model = nn.Sequential(nn.Linear(32, 16), GroupedExperts())
    mod = LowPrecisionTrainingModifier(scheme={"fp8_block_e4m3": ["Linear"], "fp8_block_e5m2": ["GroupedExperts"]}, lora_rank=0)
    assert mod.convert(model) is True
    assert isinstance(model[0].weight.data, Wrapped) and not isinstance(model[0].bias.data, Wrapped)
    assert model[1].w1.data.config.precision == "fp8_block_e5m2" and model[0].weight.data.config == config()
