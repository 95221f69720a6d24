"""How the MXFP8 linears behind a norm may be called: by keyword, and refused on host tensors like the other calls."""
import pytest
import torch

from alto_b200 import norm


@pytest.mark.parametrize("weights", [torch.zeros(64, 128), [torch.zeros(64, 128)], []])
def test_host_tensors_are_refused_by_name(weights):
    x, nw = torch.zeros(32, 128), torch.ones(128)
    for call in (lambda: norm.rms_norm_mxfp8_linear(x, nw, weights), lambda: norm.rms_norm_mxfp8_linear(x, nw, weights, residual=x),
                 lambda: norm.rms_norm_mxfp8_linear(x=x, norm_weight=nw, weights=weights)):
        with pytest.raises(RuntimeError, match="rms_norm_mxfp8_linear runs on CUDA tensors only"):
            call()


def test_arguments_by_keyword_reach_the_call(monkeypatch):
    seen = []
    monkeypatch.setattr(norm, "_check", lambda name, x, weight, residual, eps: seen.append((name, x, weight, residual, eps)))
    x, nw = torch.zeros(32, 128), torch.ones(128)
    with pytest.raises(ValueError, match="e3m4"):
        norm.rms_norm_mxfp8_linear(weights=torch.zeros(64, 128), residual=x, x=x, eps=1e-6, norm_weight=nw, fp8_variant="e3m4")
    assert seen[0][0] == "rms_norm_mxfp8_linear" and seen[0][1] is x and seen[0][2] is nw and seen[0][4] == 1e-6

