"""SwiGLU whose input is kept in 8 bits: forward bit for bit that of ``swiglu``, codes those of ``convert_to_mxfp8``, the gradient
that of the activation at the codes' values, in 64 bits.

Tolerance of a gradient: half a step of bf16 (2^-8 of itself) and what fp32 leaves of its terms: the sigmoid is off by four
steps, products and the sum 1 + g (1 - s) by half a step each: below 16 2^-24 = 2^-20 of |go u| s (1 + |g|) and |go g| s."""
import gc

import pytest
import torch

from alto_b200 import _lib as L
from alto_b200 import mxfp8
from alto_b200.swiglu import swiglu

pytestmark = pytest.mark.gpu


def _h(rows, hidden, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, 2 * hidden, generator=g, device="cuda") * std).bfloat16(), torch.randn(rows, hidden, generator=g, device="cuda").bfloat16()


def _value64(v, dy):
    n = v.shape[1] // 2
    return (v[:, :n] * torch.sigmoid(v[:, :n]) * v[:, n:] * dy.double()).sum()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows, hidden", [(1, 32), (3, 96), (128, 64), (37, 2880), (5, 14336), (700, 1056), (0, 64)])
@pytest.mark.parametrize("std", [1.0, 20.0, 1e-20])
def test_forward_codes_and_gradient(rows, hidden, fmt, std):
    h, dy = _h(rows, hidden, std=std)
    leaf = h.clone().requires_grad_(True)
    y = swiglu(leaf, checkpoint=fmt)
    assert torch.equal(y.detach(), swiglu(h)) and torch.equal(swiglu(h, checkpoint=fmt), y.detach())
    (dh,) = torch.autograd.grad(y, leaf, dy)
    if rows == 0:
        assert dh.shape == h.shape
        return
    out, codes, scales = L.swiglu_keep_forward(h, {"e4m3": L.FMT_MXFP8_E4M3, "e5m2": L.FMT_MXFP8_E5M2}[fmt])
    want = mxfp8.convert_to_mxfp8(h, mxfp_format=fmt)
    assert torch.equal(codes, want[0].view(torch.uint8)) and torch.equal(scales, want[1])
    v = mxfp8.convert_from_mxfp8(*want).double()
    g, u, d = v[:, :hidden], v[:, hidden:], dy.double()
    s = torch.sigmoid(g)
    exact = torch.cat([d * u * s * (1 + g * (1 - s)), d * g * s], 1)
    size = torch.cat([(d * u * s * (1 + g.abs())).abs(), (d * g * s).abs()], 1)
    assert ((dh.double() - exact).abs() <= exact.abs() * 2.0 ** -8 + size * 2.0 ** -20 + 1e-37).all()


def test_forward_of_every_bf16_gate_is_that_of_the_other_kernel():
    # the two kernels evaluate SiLU by different instructions; rounded to bf16 they agree for each of the 65536 gates
    gates = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).cuda().view(2048, 32)
    for up in (1.0, -3.015625, 1e30):
        h = torch.cat([gates, torch.full_like(gates, up)], 1)
        leaf = h.clone().requires_grad_(True)
        got, want = swiglu(leaf, checkpoint="e4m3").detach(), swiglu(h)
        same = (got.view(torch.int16) == want.view(torch.int16)) | (torch.isnan(got) & torch.isnan(want))
        assert same.all(), [(g, a, b) for g, a, b in zip(gates[~same].tolist(), got[~same].tolist(), want[~same].tolist())][:20]


def test_gradient_against_differences():
    h, dy = _h(11, 64)
    leaf = h.clone().requires_grad_(True)
    (dh,) = torch.autograd.grad(swiglu(leaf, checkpoint="e4m3"), leaf, dy)
    v, step = mxfp8.convert_from_mxfp8(*mxfp8.convert_to_mxfp8(h)).double(), 1e-4
    for seed in range(4):
        way = torch.randn(11, 128, generator=torch.Generator().manual_seed(seed)).double().cuda()
        along = (_value64(v + step * way, dy) - _value64(v - step * way, dy)) / (2 * step)
        # every entry of dh is off by at most 2^-8 of itself
        assert abs((dh.double() * way).sum() - along) <= 2.0 ** -8 * (dh.double() * way).abs().sum() + 1e-6


def test_infinities_nan_and_zero_rows_stay_in_their_blocks():
    h, dy = _h(8, 128)
    h[0] = 0
    h[1, 5], h[2, 200] = float("nan"), float("inf")
    leaf = h.clone().requires_grad_(True)
    y = swiglu(leaf, checkpoint="e5m2")
    assert torch.equal(y.detach().view(torch.int16), swiglu(h).view(torch.int16))
    (dh,) = torch.autograd.grad(y, leaf, dy)
    assert (dh[0] == 0).all() and torch.isfinite(dh[3:]).all()
    assert torch.isfinite(dh[1, 32:128]).all() and torch.isfinite(dh[2, :64]).all()


def test_columns_of_a_wider_buffer_and_gradients_without_strides():
    wide, _ = _h(20, 96)
    leaf = wide.clone().requires_grad_(True)
    swiglu(leaf[:, 64:192], checkpoint="e4m3").sum().backward()
    again = wide[:, 64:192].clone().requires_grad_(True)
    swiglu(again, checkpoint="e4m3").backward(torch.ones(20, 64, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(leaf.grad[:, 64:192], again.grad) and (leaf.grad[:, :64] == 0).all()


def test_h_is_not_held_between_the_passes():
    gc.collect()
    scale = torch.ones((), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    base = torch.randn(4096, 4096, device="cuda").bfloat16()
    held = {}
    for checkpoint in (None, "e4m3"):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = swiglu(base + scale, checkpoint=checkpoint)
        held[checkpoint] = torch.cuda.memory_allocated() - before - y.numel() * 2
        del y
    assert held[None] >= 2 * base.numel() and held["e4m3"] <= 1.04 * base.numel()


def test_captured_step_replays_on_new_contents():
    h, dy = _h(256, 512)
    leaf = h.clone().requires_grad_(True)

    def step():
        y = swiglu(leaf, checkpoint="e4m3")
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    h2, dy2 = _h(256, 512, 7)
    with torch.no_grad():
        leaf.copy_(h2), dy.copy_(dy2)
    graph.replay()
    got = [t.clone() for t in out]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
