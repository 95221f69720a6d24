"""Refusals of the norm, routing, row plan and SwiGLU calls that need no device."""
import pytest
import torch

from alto_b200 import _lib as L
from alto_b200 import norm, routing, swiglu


def test_no_call_takes_host_tensors():
    x, w = torch.zeros(4, 64), torch.ones(64)
    for call in (lambda: norm.rms_norm(x, w), lambda: norm.rms_norm_mxfp8(x, w), lambda: norm.rms_norm(x, w, residual=x),
                 lambda: routing.route_experts(x, 2), lambda: routing.expert_plan(torch.zeros(4, 2, dtype=torch.int32), 8),
                 lambda: swiglu.swiglu(torch.zeros(4, 64, dtype=torch.bfloat16), checkpoint="e4m3")):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_swiglu_refuses_unknown_formats_and_blocks_that_do_not_fit():
    h = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="checkpoint format"):
        swiglu.swiglu(h, checkpoint="int8")
    with pytest.raises(ValueError, match="multiple of 32"):
        swiglu.swiglu(h[:, :32], checkpoint="e4m3")
    with pytest.raises(TypeError):
        swiglu.swiglu(h.float(), checkpoint="e4m3")


def _norm_args(**change):
    # addresses that nothing reads: every call below is refused before a launch
    a = L.RmsNormArgs(4, 64, 64, 0, 256, None, 256, 256, None, None, None, None, 1e-5, L.DT_BF16, L.DT_BF16, -1)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change, status", [
    (dict(cols=0), L.E_SHAPE), (dict(rows=-1), L.E_SHAPE), (dict(ld_x=63), L.E_SHAPE), (dict(x=None), L.E_SHAPE),
    (dict(residual=256), L.E_SHAPE), (dict(normed_out=256), L.E_SHAPE), (dict(dtype=7), L.E_UNSUPPORTED), (dict(weight_dtype=2), L.E_UNSUPPORTED),
    (dict(format=L.FMT_NVFP4), L.E_UNSUPPORTED), (dict(format=L.FMT_MXFP8_E4M3), L.E_SHAPE),
    (dict(format=L.FMT_MXFP8_E4M3, scale_plain=256, cols=48, ld_x=64), L.E_SHAPE), (dict(rows=2 ** 31), L.E_LIMIT)])
def test_norm_entry_point_refuses(change, status):
    assert L.lib().altob200_rms_norm_forward(_norm_args(**change), None) == status


def test_norm_entry_point_takes_no_rows():
    assert L.lib().altob200_rms_norm_forward(_norm_args(rows=0), None) == 0
    assert L.lib().altob200_rms_norm_forward(None, None) == L.E_SHAPE
    assert L.lib().altob200_rms_norm_backward(None, None, None) == L.E_SHAPE


@pytest.mark.parametrize("change, status", [
    (dict(ld_grad=63), L.E_SHAPE), (dict(grad_in=None), L.E_SHAPE), (dict(dtype=5), L.E_UNSUPPORTED),
    (dict(grad_stream=256, ld_grad_stream=8), L.E_SHAPE), (dict(grad_weight=256), L.E_SHAPE), (dict(rows=2 ** 31), L.E_LIMIT)])
def test_norm_gradient_entry_point_refuses(change, status):
    a = L.RmsNormGradArgs(4, 64, 64, 64, 0, 256, 256, None, 256, 256, None, 1e-5, L.DT_F32, L.DT_F32)
    for k, v in change.items():
        setattr(a, k, v)
    assert L.lib().altob200_rms_norm_backward(a, None, None) == status


def _route_params(**change):
    p = L.RouteParams(L.DT_F32, 64, 4, 0, 1, 1, 1, 1, 1.0)
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change, status", [
    (dict(experts=513), L.E_LIMIT), (dict(top_k=17), L.E_LIMIT), (dict(num_groups=33), L.E_LIMIT), (dict(top_k=0), L.E_SHAPE),
    (dict(num_groups=5), L.E_SHAPE), (dict(num_groups=4, groups_kept=5), L.E_SHAPE), (dict(group_top=3), L.E_SHAPE),
    (dict(num_groups=32, groups_kept=1, top_k=3), L.E_SHAPE), (dict(dtype=9), L.E_UNSUPPORTED)])
def test_route_entry_point_refuses(change, status):
    assert L.lib().altob200_route_forward(_route_params(**change), 256, 8, 64, None, 256, 256, None) == status


def test_route_entry_point_refuses_rows_that_overlap():
    assert L.lib().altob200_route_forward(_route_params(), 256, 8, 63, None, 256, 256, None) == L.E_SHAPE
    assert L.lib().altob200_route_backward(_route_params(), 256, 8, 63, 256, 256, 256, None) == L.E_SHAPE
    assert L.lib().altob200_route_forward(_route_params(), None, 0, 64, None, None, None, None) == 0


@pytest.mark.parametrize("args, status", [
    ((256, 16, 8, 2, 8, 128, 64), L.E_UNSUPPORTED), ((256, 32, 8, 2, 1025, 128, 64), L.E_LIMIT), ((256, 32, -1, 2, 8, 128, 64), L.E_SHAPE),
    ((256, 32, 8, 0, 8, 128, 64), L.E_SHAPE), ((256, 32, 8, 2, 8, 0, 64), L.E_SHAPE), ((None, 32, 8, 2, 8, 128, 64), L.E_SHAPE),
    ((256, 32, 2 ** 30, 4, 8, 128, 64), L.E_LIMIT), ((256, 32, 8, 2, 8, 128, 2 ** 31), L.E_LIMIT),
    ((256, 32, 4096, 4, 8, 128, 64), L.E_SHAPE)])   # the last: no work space where one is needed
def test_plan_entry_point_refuses(args, status):
    assert L.lib().altob200_expert_plan(*args, 256, 256, 256, 256, 256, None, None) == status


@pytest.mark.parametrize("args, status", [
    ((4, 32, 64, L.FMT_NVFP4), L.E_UNSUPPORTED), ((4, 48, 96, L.FMT_MXFP8_E4M3), L.E_SHAPE), ((4, 32, 60, L.FMT_MXFP8_E4M3), L.E_SHAPE),
    ((-1, 32, 64, L.FMT_MXFP8_E4M3), L.E_SHAPE), ((4, 32, 68, L.FMT_MXFP8_E4M3), L.E_ALIGN)])
def test_swiglu_entry_points_refuse(args, status):
    assert L.lib().altob200_swiglu_keep_forward(256, *args, 256, 256, 256, None) == status
