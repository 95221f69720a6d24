"""SwiGLU of an expert MLP whose gate and up projections are one grouped GEMM: ``swiglu(h)`` with
``h = [gate | up]`` equals ``silu(h[:, :H]) * h[:, H:]`` (same bf16 roundings, forward and backward)
in one kernel per direction instead of eight tensor-op passes over the routed rows.

``swiglu(h, checkpoint="e4m3")`` returns the same and keeps ``h`` for the backward pass as MXFP8 codes and scales
(``convert_to_mxfp8`` of it, written from the same read) instead of bf16: 1.03 bytes an element for 2 between the two
passes, once nothing else holds ``h``.  Its gradient is that of the activation at the values of the codes, computed in fp32.

The module that owns this activation in the reference's setting is ``GroupedExperts`` of its
TorchTitan fork, whose parameters the modifier swaps (alto/modifiers/lpt/base.py:186-187); the
grouped GEMMs on either side are ``alto_b200.grouped``."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["swiglu"]

_KEEP = {"e4m3": _lib.FMT_MXFP8_E4M3, "e5m2": _lib.FMT_MXFP8_E5M2}


def _packed(t: torch.Tensor) -> torch.Tensor:
    """Contiguous rows from a 16-byte boundary, as the kernels' vectors need them."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h):
        h = _packed(h)
        ctx.save_for_backward(h)
        return _lib.swiglu_forward(h)

    @staticmethod
    def backward(ctx, grad_out):
        (h,) = ctx.saved_tensors
        return _lib.swiglu_backward(h, _packed(grad_out))


class _SwiGLUKept(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, fmt):
        out, codes, scales = _lib.swiglu_keep_forward(_packed(h), fmt)
        ctx.save_for_backward(codes, scales)
        ctx.fmt = fmt
        return out

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, grad_out):
        codes, scales = ctx.saved_tensors
        return _lib.swiglu_kept_backward(codes, scales, _packed(grad_out), ctx.fmt), None


def swiglu(h: torch.Tensor, checkpoint: Optional[str] = None) -> torch.Tensor:
    """h: [rows, 2H] bf16 on a CUDA device, H a multiple of 8 -> [rows, H].  ``checkpoint``: None, or the 8-bit format
    ("e4m3", "e5m2") in which h is kept for the backward pass; H is then a multiple of 32."""
    if h.dim() != 2 or h.shape[1] % 16 != 0:
        raise ValueError(f"swiglu expects [rows, 2H] with H a multiple of 8, got {tuple(h.shape)}")
    if h.dtype != torch.bfloat16:
        raise TypeError(f"swiglu expects bfloat16, got {h.dtype}")
    if checkpoint is None:
        return _SwiGLU.apply(h)
    if checkpoint not in _KEEP:
        raise ValueError(f"unsupported checkpoint format {checkpoint!r}; supported: {sorted(_KEEP)}")
    if h.shape[1] % 64 != 0:
        raise ValueError(f"an 8-bit checkpoint expects [rows, 2H] with H a multiple of 32, got {tuple(h.shape)}")
    if not h.is_cuda:
        raise RuntimeError("swiglu runs on CUDA tensors only (no CPU fallback)")
    if not (h.requires_grad and torch.is_grad_enabled()):
        return _SwiGLU.apply(h)      # nothing to keep
    return _SwiGLUKept.apply(h, _KEEP[checkpoint])
