"""What the FP8 block operators and gradient clipping refuse before anything is launched, on the CPU."""
import math

import pytest
import torch

from alto_b200 import fp8_block as FB
from alto_b200 import grad_clip as GC
from alto_b200 import grouped


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(16, 32, dtype=torch.bfloat16)
    codes, scales = w.to(torch.float8_e4m3fn), torch.ones(1, 1)
    offs = torch.tensor([4], dtype=torch.int32)
    for call in (lambda: FB.convert_to_fp8_block(x), lambda: FB.convert_from_fp8_block(codes, torch.ones(16, 1)),
                 lambda: FB.blockwise_fp8_gemm(codes, torch.ones(16, 1), codes, torch.ones(16, 1)),
                 lambda: FB.fp8_block_linear(x, codes, scales), lambda: FB._to_fp8_block_then_scaled_mm(x, w),
                 lambda: FB.fp8_block_grouped_linear(x, codes[None], scales[None], offs),
                 lambda: grouped._quantize_then_fp8_block_scaled_grouped_mm(x, w.t()[None], offs=offs),
                 lambda: GC.grad_norm([x]), lambda: GC.clip_grads([x], 1.0)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_what_is_not_a_tensor():
    for bad in ([None], [1.0]):
        for call in (lambda: GC.grad_norm(bad), lambda: GC.clip_grads(bad, 1.0)):
            with pytest.raises(TypeError, match="expects tensors"):
                call()


def test_norms_and_lists():
    assert float(GC.grad_norm([])) == 0.0 and float(GC.clip_grads([], 1.0)) == 0.0
    assert float(GC.clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0
    for p in (1.0, 0.0, -2.0, 3.0):
        with pytest.raises(ValueError, match="norms are 2 and inf"):
            GC.grad_norm([], p)
    assert GC._kind(math.inf) and GC._kind("inf") and not GC._kind(2)
