"""Root-mean-square norm of token rows, with the residual's addition in front of it.

    rms_norm(x, weight, eps)                      y = x / sqrt(mean(x^2) + eps) * weight
    rms_norm(x, weight, eps, residual=res)        (y, r): r = x + res in the type of x, y the norm of r
    rms_norm_mxfp8(...)                           y as MXFP8 codes and block scales (``convert_to_mxfp8`` of y, bit for bit)

One kernel each, one read of the rows; sums are fp32 and y is rounded once.  ``rms_norm`` is differentiable in x, residual
and weight (one pass for the rows' gradient, which x and the residual share, and a short one that joins the weight's).
The codes of ``rms_norm_mxfp8`` go into ``mxfp8.blockwise_mxfp8_gemm`` or, in a training step, through
``rms_norm_mxfp8_linear`` into the MXFP8 linear.

The decoder blocks that the reference converts have this norm in front of their linears
(alto/modifiers/lpt/base.py:171-192); its kernels leave it to tensor operations."""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from . import _lib as L
from . import _linear as E
from .nvfp4 import unwrap_weight_wrapper

__all__ = ["rms_norm", "rms_norm_mxfp8", "rms_norm_mxfp8_linear"]

_FP8 = {"e4m3": (L.FMT_MXFP8_E4M3, torch.float8_e4m3fn), "e5m2": (L.FMT_MXFP8_E5M2, torch.float8_e5m2)}
_TYPES = (torch.bfloat16, torch.float32)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[rows, cols] view (or copy) whose rows are contiguous and do not overlap."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    elif t.is_contiguous() and t.shape[0] > 1 and t.shape[1] > 1:      # the usual case, with the fewest questions
        return t
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:      # one column or one row: strides that say nothing
        t = t.as_strided(t.shape, (t.shape[1], 1))
    return t


def _check(name: str, x, weight, residual, eps) -> None:
    # one pass over what is usual; what is not is told apart below
    if (x.is_cuda and x.dtype in _TYPES and weight.dtype in _TYPES and weight.shape == x.shape[-1:] and weight.device == x.device
            and eps >= 0.0 and x.dim() > 0 and x.shape[-1] > 0
            and (residual is None or (residual.shape == x.shape and residual.dtype is x.dtype and residual.device == x.device))):
        return
    if not x.is_cuda or not weight.is_cuda or (residual is not None and not residual.is_cuda):
        raise RuntimeError(f"{name} runs on CUDA tensors only (no CPU fallback)")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} expects rows in the last dimension, got {tuple(x.shape)}")
    if x.dtype not in _TYPES or weight.dtype not in _TYPES:
        raise TypeError(f"{name} expects bfloat16 or float32, got {x.dtype} and a weight of {weight.dtype}")
    if weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"{name} expects a weight of [{x.shape[-1]}], got {tuple(weight.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{name} expects a residual like x ({tuple(x.shape)}, {x.dtype}), got {tuple(residual.shape)}, "
                         f"{residual.dtype}")
    if weight.device != x.device or (residual is not None and residual.device != x.device):
        raise ValueError(f"{name} expects all tensors on one device")
    raise ValueError(f"{name} expects eps >= 0, got {eps}")


@L.traced("rms_norm")
def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """Norm of the rows of x [..., cols] (bf16 or fp32; weight [cols] in either type).  With ``residual`` (like x) returns
    (y, r), r = x + residual rounded to the type of x and y the norm of r; else y."""
    _check("rms_norm", x, weight, residual, eps)
    host = L._autograd_module or L.autograd()
    return host.rms_norm(x, weight, eps) if residual is None else host.rms_norm_residual(x, weight, residual, eps)


@L.traced("rms_norm_mxfp8")
def rms_norm_mxfp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: Optional[torch.Tensor] = None,
                   mxfp_format: str = "e4m3"):
    """The norm's result as MXFP8: (codes [..., cols], scales uint8 [..., cols / 32]), and r behind them with ``residual``.
    cols is a multiple of 32.  Codes and scales are those of ``convert_to_mxfp8(rms_norm(...))``.  Not differentiable, as
    the quantizers are not: for evaluation and serving."""
    _check("rms_norm_mxfp8", x, weight, residual, eps)
    if mxfp_format not in _FP8:
        raise ValueError(f"Unsupported FP8 format: {mxfp_format}. Supported: {sorted(_FP8)}")
    if x.shape[-1] % 32 != 0:
        raise ValueError(f"rms_norm_mxfp8 expects rows of a multiple of 32, got {x.shape[-1]}")
    fmt, dtype = _FP8[mxfp_format]
    codes, stream, scales = L.rms_norm_forward(_rows(x), weight if weight.is_contiguous() else weight.contiguous(), eps,
                                               None if residual is None else _rows(residual), fmt)
    codes = codes.view(dtype)
    if x.dim() != 2:
        codes, scales = codes.view(x.shape), scales.view(*x.shape[:-1], x.shape[-1] // 32)
        stream = None if stream is None else stream.view(x.shape)
    return (codes, scales) if stream is None else (codes, scales, stream)


class _RMSNormMXFP8Linear(torch.autograd.Function):
    """The norm and the MXFP8 linears behind it.  Forward writes the operand of the forward products straight from the
    norm; what is kept is the stream and the codes of the backward products, no bf16 norm.  Results have two dimensions: views
    made in here could not be written to."""

    @staticmethod
    def forward(ctx, x, norm_weight, residual, eps, fmt, use_2dblock_w, *weights):
        x2 = _rows(x)
        M, K = x2.shape
        weights = [unwrap_weight_wrapper(w) for w in weights]
        for w in weights:
            torch._check(w.dim() == 2 and w.shape[1] == K, lambda: f"linear weights must be [N, {K}], got {tuple(w.shape)}")
            torch._check(w.dtype == x.dtype, lambda: f"weight dtype ({w.dtype}) must match x dtype ({x.dtype})")
            E.check_dims("rms_norm_mxfp8_linear", M, K, w.shape[0])
        need_w = ctx.needs_input_grad[6:]
        need_y = any(ctx.needs_input_grad[:3])
        y = torch.empty(M, K, dtype=x.dtype, device=x.device) if any(need_w) else None
        codes, stream, scales = L.rms_norm_forward(x2, norm_weight.contiguous(), eps, None if residual is None else _rows(residual),
                                                   fmt, packed=True, normed=y)
        x_k = E.Operand(codes, scales, None, M, K, fmt)
        x_m = None if y is None else E.quant_cols(y, fmt, None, None, E.RTN)
        outs, saved = [], []
        for w in weights:
            w2 = w if isinstance(w, E.PrequantizedWeight) else E.as_2d_rows(w.detach())
            w_k, w_t = E.weight_operands(w2, fmt, use_2dblock_w=use_2dblock_w, use_outer_scale=False,
                                         want_t=need_y)
            outs.append(E.gemm(x_k, w_k, x.dtype))
            saved += [None, None] if w_t is None else [w_t.codes, w_t.scales]
        ctx.save_for_backward(x if stream is None else stream, norm_weight,
                              *([None, None] if x_m is None else [x_m.codes, x_m.scales]), *saved)
        ctx.dims, ctx.shape, ctx.eps, ctx.fmt, ctx.outs = (M, K), x.shape, eps, fmt, [w.shape[0] for w in weights]
        ctx.set_materialize_grads(False)
        return tuple(outs) if stream is None else (*outs, stream)

    @staticmethod
    @L.once_differentiable
    def backward(ctx, *grads):
        stream, norm_weight, xc, xs, *wt = ctx.saved_tensors
        (M, K), fmt = ctx.dims, ctx.fmt
        n = len(ctx.outs)
        grad_stream = grads[n] if len(grads) > n else None
        need_x, need_nw, need_res = ctx.needs_input_grad[:3]
        dy, dws = None, []
        for i, N in enumerate(ctx.outs):
            g = grads[i]
            dw = None
            if g is not None:
                g2 = E.as_2d_rows(g)
                if need_x or need_nw or need_res:
                    g_n = E.quant_rows(g2, fmt, None, E.RTN)
                    part = E.gemm(g_n, E.Operand(wt[2 * i], wt[2 * i + 1], None, K, N, fmt), g.dtype)
                    dy = part if dy is None else dy + part
                if ctx.needs_input_grad[6 + i]:
                    g_m = E.quant_cols(g2, fmt, None, None, E.RTN)
                    dw = E.gemm(g_m, E.Operand(xc, xs, None, K, M, fmt), g.dtype)
            elif ctx.needs_input_grad[6 + i]:
                dw = torch.zeros(N, K, dtype=stream.dtype, device=stream.device)
            dws.append(dw)
        gx, gw = grad_stream, None
        if dy is not None:
            gx, gw = L.rms_norm_backward(dy, _rows(stream), norm_weight.contiguous(), ctx.eps,
                                         None if grad_stream is None else _rows(grad_stream), need_nw)
        elif need_nw:
            gw = torch.zeros_like(norm_weight)
        gx = None if gx is None else gx.reshape(ctx.shape)
        return (gx if need_x else None, gw, gx if need_res else None, None, None, None, *dws)


@L.on_device_of
def _linears(x, norm_weight, residual, eps, fmt, use_2dblock_w, weights):
    return _RMSNormMXFP8Linear.apply(x, norm_weight, residual, eps, fmt, use_2dblock_w, *weights)


@L.traced("rms_norm_mxfp8_linear")
def rms_norm_mxfp8_linear(x: torch.Tensor, norm_weight: torch.Tensor, weights: Union[torch.Tensor, Sequence[torch.Tensor]],
                          eps: float = 1e-5, residual: Optional[torch.Tensor] = None, fp8_variant: str = "e4m3",
                          use_2dblock_w: bool = False):
    """The norm of x (behind the residual's addition) through one MXFP8 linear or several that read the same norm (query, key
    and value; gate and up): what ``_to_mxfp8_then_scaled_mm(rms_norm(x, norm_weight, eps, residual), w, fp8_variant,
    False, False, use_2dblock_w)`` computes for each, bit for bit.  The forward products read codes that the norm writes; where a
    weight requires a gradient the norm is written in the type of x too, for the quantizer of that gradient's operand, and
    not kept.

    ``weights``: one [N, K] or a sequence of them.  Returns the outputs in their order (one tensor for one weight), and r
    behind them with ``residual``.  Differentiable in x, residual, norm_weight and weights; gradients that several linears send
    to the norm are added in the type of x, in their order.  Tokens, K and N are multiples of 32, as everywhere in the
    MXFP8 linear."""
    many = not isinstance(weights, torch.Tensor)
    weights = tuple(weights) if many else (weights,)
    _check("rms_norm_mxfp8_linear", x, norm_weight, residual, eps)
    if fp8_variant not in _FP8:
        raise ValueError(f"Unsupported FP8 variant: {fp8_variant}. Supported: {sorted(_FP8)}")
    if not weights or any(w.device != x.device for w in weights):
        raise ValueError("rms_norm_mxfp8_linear expects weights on the device of x")
    if not torch.is_grad_enabled() and not L.forward_mode():      # an evaluation pass: its parameters still say that they require gradients
        x, norm_weight = x.detach(), norm_weight.detach()
        residual = None if residual is None else residual.detach()
        weights = tuple(w.detach() if type(w) is torch.nn.Parameter or type(w) is torch.Tensor else
                        unwrap_weight_wrapper(w).detach() for w in weights)
    got = _linears(x, norm_weight, residual, eps, _FP8[fp8_variant][0], bool(use_2dblock_w), weights)
    if x.dim() != 2:
        got = tuple(t.view(*x.shape[:-1], t.shape[1]) for t in got)
    if not many and residual is None:
        return got[0]
    return got
