"""FP8 with one fp32 scale for each block of 128: quantizers, the product, and linears dense and grouped by expert, on B200.

    convert_to_fp8_block / convert_from_fp8_block      codes and scales along an axis, or of squares of 128 x 128
    blockwise_fp8_gemm(a, a_s, b, b_s)                 a b^T of two quantised operands
    _to_fp8_block_then_scaled_mm / FP8BlockLinearFunction            a training step's linear (x in blocks of a row, weights
                                                                     in squares; the weight gradient in blocks of tokens)
    fp8_block_linear / fp8_block_grouped_linear        serving: weights that are there as codes and scales, from one token up

A block's scale is max(|largest|, 1e-12) / top (top: 448 for E4M3, 57344 for E5M2) and its codes are the quotients by it, to
nearest; a last block is as short as the dimension.  The products of a block of 128 are summed by the tensor cores and added
up in fp32 with both scales.  Features (in and out) are multiples of 16, tokens any number.  The grouped training form is
``grouped._quantize_then_fp8_block_scaled_grouped_mm``.

The reference has this format in a part that its recipes do not reach (alto/kernels/blockwise_fp8/blockwise_linear.py:161);
recipes name it here as the scheme "fp8_block" (``dispatch.TrainingOpConfig``, ``lpt.LowPrecisionTrainingModifier``)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib as L
from .nvfp4 import outside_of_grad_mode, unwrap_weight_wrapper

__all__ = ["convert_to_fp8_block", "convert_from_fp8_block", "blockwise_fp8_gemm", "FP8BlockLinearFunction", "fp8_block_linear",
           "fp8_block_grouped_linear"]

BLOCK_SIZE = 128
SUPPORTED_FORMATS = ["e4m3", "e5m2"]
_FMT = {"e4m3": L.FMT_MXFP8_E4M3, "e5m2": L.FMT_MXFP8_E5M2}
_CODE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FMT_OF_DTYPE = {torch.float8_e4m3fn: L.FMT_MXFP8_E4M3, torch.float8_e5m2: L.FMT_MXFP8_E5M2}
_TYPES = (torch.bfloat16, torch.float32)


def _blocks(n: int) -> int:
    return (n + BLOCK_SIZE - 1) // BLOCK_SIZE


def _rows(x: torch.Tensor) -> torch.Tensor:
    """[rows, cols] view (or copy) with unit column stride, rows that do not overlap and begin on 16 bytes."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.shape[0] <= 1:
        if x2.stride(1) == 1 and x2.data_ptr() % 16 == 0:
            return x2
    elif x2.stride(1) == 1 and x2.stride(0) >= x2.shape[1] and x2.stride(0) * x2.element_size() % 16 == 0 and x2.data_ptr() % 16 == 0:
        return x2
    return x2.clone(memory_format=torch.contiguous_format)


def _packed(t: torch.Tensor) -> torch.Tensor:
    """Without gaps and from a 16-byte boundary."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_format(fmt: str) -> None:
    if fmt not in SUPPORTED_FORMATS:
        raise ValueError(f"Unsupported FP8 format: {fmt}. Supported: {SUPPORTED_FORMATS}")


# ---------------------------------------------------------------------------------------------
# quantizers
# ---------------------------------------------------------------------------------------------
@L.traced("convert_to_fp8_block")
def convert_to_fp8_block(data_hp: torch.Tensor, block_size: int = BLOCK_SIZE, fp8_format: str = "e4m3", axis: int = -1,
                         is_2d_block: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes like ``data_hp``, fp32 scales) of a tensor [..., M, N] (bf16 or fp32), N a multiple of 16.  Scales are
    [..., M, ceil(N / 128)] along ``axis`` -1, [..., ceil(M / 128), N] along -2 and [..., ceil(M / 128), ceil(N / 128)] for
    ``is_2d_block`` (M a multiple of 16 too).  Along -2 the codes are a view of a tensor that has that axis last."""
    if not data_hp.is_cuda:
        raise RuntimeError("alto_b200 quantizers run on CUDA tensors only (no CPU fallback)")
    _check_format(fp8_format)
    if block_size != BLOCK_SIZE:
        raise ValueError(f"FP8 block kernels are built for block_size {BLOCK_SIZE}, got {block_size}")
    if data_hp.dtype not in _TYPES:
        raise TypeError(f"convert_to_fp8_block expects bfloat16 or float32, got {data_hp.dtype}")
    if data_hp.dim() < 2 or data_hp.shape[-1] % 16 != 0 or data_hp.shape[-1] == 0:
        raise ValueError(f"convert_to_fp8_block expects [..., M, N] with N a multiple of 16, got {tuple(data_hp.shape)}")
    axis = axis if axis < 0 else axis - data_hp.dim()
    if axis not in (-1, -2):
        raise ValueError(f"axis must address one of the last two dimensions, got {axis}")
    fmt, lead, (M, N) = _FMT[fp8_format], data_hp.shape[:-2], data_hp.shape[-2:]
    x = data_hp.detach()
    if is_2d_block:
        if M % 16 != 0 or M == 0:
            raise ValueError(f"convert_to_fp8_block expects rows of 2-D blocks in multiples of 16, got {tuple(data_hp.shape)}")
        codes, codes_t, scales = L.fp8_block_quantize_squares(_packed(x).view(-1, M, N), fmt, axis == -1, axis == -2)
        codes = codes.view(*lead, M, N) if axis == -1 else codes_t.view(*lead, N, M).transpose(-1, -2)
        return codes.view(_CODE[fp8_format]), scales.view(*lead, *scales.shape[1:])
    if axis == -1:
        (codes, scales), _ = L.fp8_block_quantize(_rows(x), fmt, True, False)
        return codes.view(data_hp.shape).view(_CODE[fp8_format]), scales.t().reshape(*lead, M, scales.shape[0])
    x3 = x.reshape(-1, M, N)
    parts = [L.fp8_block_quantize(_rows(m), fmt, False, True)[1] for m in x3]
    if not parts:
        codes = torch.empty(0, N, _blocks(M) * BLOCK_SIZE, dtype=torch.uint8, device=x.device)
        scales = torch.empty(0, _blocks(M), N, dtype=torch.float32, device=x.device)
    elif len(parts) == 1:
        codes, scales = parts[0][0].unsqueeze(0), parts[0][1].unsqueeze(0)
    else:
        codes, scales = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    codes = codes[..., :M].unflatten(0, lead).transpose(-1, -2) if lead else codes[0, :, :M].t()
    return codes.view(_CODE[fp8_format]), scales.view(*lead, *scales.shape[1:])


@L.traced("convert_from_fp8_block")
def convert_from_fp8_block(data_lp: torch.Tensor, scales: torch.Tensor, output_dtype: torch.dtype = torch.float32,
                           block_size: int = BLOCK_SIZE, axis: int = -1, is_2d_block: bool = False) -> torch.Tensor:
    """Values of what ``convert_to_fp8_block`` returned, codes [..., M, N] with N a multiple of 8."""
    if not data_lp.is_cuda or not scales.is_cuda:
        raise RuntimeError("alto_b200 dequantizers run on CUDA tensors only (no CPU fallback)")
    if data_lp.dtype not in _FMT_OF_DTYPE:
        raise ValueError(f"Unsupported FP8 dtype: {data_lp.dtype}")
    if block_size != BLOCK_SIZE:
        raise ValueError(f"FP8 block kernels are built for block_size {BLOCK_SIZE}, got {block_size}")
    if output_dtype not in _TYPES:
        raise TypeError(f"convert_from_fp8_block writes bfloat16 or float32, not {output_dtype}")
    if data_lp.dim() < 2 or data_lp.shape[-1] % 8 != 0:
        raise ValueError(f"convert_from_fp8_block expects [..., M, N] with N a multiple of 8, got {tuple(data_lp.shape)}")
    axis = axis if axis < 0 else axis - data_lp.dim()
    if axis not in (-1, -2):
        raise ValueError(f"axis must address one of the last two dimensions, got {axis}")
    lead, (M, N) = data_lp.shape[:-2], data_lp.shape[-2:]
    by_row, by_col = is_2d_block or axis == -2, is_2d_block or axis == -1
    want = (*lead, _blocks(M) if by_row else M, _blocks(N) if by_col else N)
    if scales.dtype != torch.float32 or tuple(scales.shape) != want or scales.device != data_lp.device:
        raise ValueError(f"convert_from_fp8_block expects fp32 scales {want} on {data_lp.device}, got {tuple(scales.shape)}, "
                         f"{scales.dtype} on {scales.device}")
    out = torch.empty(data_lp.shape, dtype=output_dtype, device=data_lp.device)
    codes, s = _packed(data_lp.detach()).view(torch.uint8), scales.detach()
    if out.numel() == 0:
        return out
    fmt = _FMT_OF_DTYPE[data_lp.dtype]
    if data_lp.dim() == 2 or (not by_row and s.is_contiguous()):      # every row has scales of its own: one matrix
        c2, s2, o2 = codes.view(-1, N), (s if s.dim() == 2 else s.view(-1, s.shape[-1])), out.view(-1, N)
        L.fp8_block_dequantize(c2, fmt, s2, s2.stride(0), s2.stride(1), 7 if by_row else 0, 7 if by_col else 0, o2)
        return out
    c3, s3, o3 = codes.view(-1, M, N), s.reshape(-1, *s.shape[-2:]), out.view(-1, M, N)
    for i in range(c3.shape[0]):
        L.fp8_block_dequantize(c3[i], fmt, s3[i], s3.stride(1), s3.stride(2), 7 if by_row else 0, 7 if by_col else 0, o3[i])
    return out


# ---------------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------------
def _row_scales(s: torch.Tensor) -> L.Fp8BlockScale:
    """Scales [chunks, rows] of blocks of a row, as the quantizer writes them."""
    return L.Fp8BlockScale(s.data_ptr(), 1, s.stride(0), 0, 0, 7)


def _square_scales(s: torch.Tensor, transposed: bool = False) -> L.Fp8BlockScale:
    """Scales [experts, rows / 128, chunks] of squares, of the matrices or of their transposes."""
    r, c = s.stride(1), s.stride(2)
    return L.Fp8BlockScale(s.data_ptr(), c if transposed else r, r if transposed else c, s.stride(0), 7, 7)


@L.traced("blockwise_fp8_gemm")
def blockwise_fp8_gemm(a: torch.Tensor, a_s: torch.Tensor, b: torch.Tensor, b_s: torch.Tensor,
                       output_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a b^T for codes a [M, K] and b [N, K] of one format with fp32 scales [M or ceil(M / 128), ceil(K / 128)] and
    [N or ceil(N / 128), ceil(K / 128)]; N and K multiples of 16."""
    if not (a.is_cuda and b.is_cuda and a_s.is_cuda and b_s.is_cuda):
        raise RuntimeError("blockwise_fp8_gemm runs on CUDA tensors only (no CPU fallback)")
    if a.dtype != b.dtype:
        raise ValueError(f"A/B FP8 dtypes must match, got a.dtype={a.dtype}, b.dtype={b.dtype}")
    if a.dtype not in _FMT_OF_DTYPE:
        raise ValueError(f"Unsupported FP8 dtype: {a.dtype}")
    if output_dtype not in _TYPES:
        raise TypeError(f"blockwise_fp8_gemm writes bfloat16 or float32, not {output_dtype}")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"blockwise_fp8_gemm expects [M, K] and [N, K], got {tuple(a.shape)} and {tuple(b.shape)}")
    (M, K), N = a.shape, b.shape[0]
    if K % 16 != 0 or N % 16 != 0 or N == 0 or K == 0:
        raise ValueError(f"blockwise_fp8_gemm expects N and K in multiples of 16, got N={N}, K={K}")
    sides = []
    for name, s, rows in (("a_s", a_s, M), ("b_s", b_s, N)):
        if s.dtype != torch.float32 or s.dim() != 2 or s.shape[1] != _blocks(K) or s.shape[0] not in (rows, _blocks(rows)):
            raise ValueError(f"blockwise_fp8_gemm expects fp32 scales {name} [{rows} or {_blocks(rows)}, {_blocks(K)}], got "
                             f"{tuple(s.shape)}, {s.dtype}")
        sides.append(L.Fp8BlockScale(s.data_ptr(), s.stride(0), s.stride(1), 0, 0 if s.shape[0] == rows else 7, 7))
    if any(t.device != a.device for t in (a_s, b, b_s)):
        raise ValueError("blockwise_fp8_gemm expects all tensors on one device")
    out = torch.empty((M, N), dtype=output_dtype, device=a.device)
    a8, b8 = _packed(a.detach()).view(torch.uint8), _packed(b.detach()).view(torch.uint8)
    L.fp8_block_gemm(a8, sides[0], b8, sides[1], out, _FMT_OF_DTYPE[a.dtype], (M, N, K))
    return out


def _product(x2: torch.Tensor, w8: torch.Tensor, sw: L.Fp8BlockScale, out: torch.Tensor, fmt: int, dims, offs=None) -> None:
    """x2 (numbers) times codes of weights; few rows an expert are quantised by the product itself."""
    M = dims[0]
    mode = 0 if offs is None else 1
    if M <= 16 * (1 if offs is None else offs.numel()):
        L.fp8_block_gemm(x2, None, w8, sw, out, fmt, dims, mode, offs)
        return
    (codes, scales), _ = L.fp8_block_quantize(x2, fmt, True, False)
    L.fp8_block_gemm(codes, _row_scales(scales), w8, sw, out, fmt, dims, mode, offs)


def _check_serving(name: str, x, w_codes, w_scales, dims: int) -> None:
    if not (x.is_cuda and w_codes.is_cuda and w_scales.is_cuda):
        raise RuntimeError(f"{name} runs on CUDA tensors only (no CPU fallback)")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name} expects bfloat16 or float32, got {x.dtype}")
    if w_codes.dtype not in _FMT_OF_DTYPE:
        raise ValueError(f"Unsupported FP8 dtype: {w_codes.dtype}")
    if w_codes.dim() != dims or x.dim() < 1 or x.shape[-1] != w_codes.shape[-1]:
        raise ValueError(f"{name} expects x [..., K] and codes [{'experts, ' if dims == 3 else ''}N, K], got {tuple(x.shape)} and "
                         f"{tuple(w_codes.shape)}")
    N, K = w_codes.shape[-2:]
    if N % 16 != 0 or K % 16 != 0 or N == 0 or K == 0:
        raise ValueError(f"{name} expects N and K in multiples of 16, got N={N}, K={K}")
    want = (*w_codes.shape[:-2], _blocks(N), _blocks(K))
    if w_scales.dtype != torch.float32 or tuple(w_scales.shape) != want:
        raise ValueError(f"{name} expects fp32 scales {want}, got {tuple(w_scales.shape)}, {w_scales.dtype}")
    if w_codes.device != x.device or w_scales.device != x.device:
        raise ValueError(f"{name} expects all tensors on one device")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError(f"{name} has no gradient: codes of weights serve evaluation")


@L.on_device_of
def _serve(x, w_codes, w_scales, offs):
    N, K = w_codes.shape[-2:]
    out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
    x2, w8 = _rows(x.detach()), _packed(w_codes.detach()).view(torch.uint8)
    s = w_scales.detach()
    _product(x2, w8, _square_scales(s if s.dim() == 3 else s.unsqueeze(0)), out, _FMT_OF_DTYPE[w_codes.dtype], (x2.shape[0], N, K), offs)
    return out


@L.traced("fp8_block_linear")
def fp8_block_linear(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor) -> torch.Tensor:
    """x W^T for x [..., K] (bf16 or fp32) and a weight that is there as codes [N, K] and fp32 scales of its squares
    [ceil(N / 128), ceil(K / 128)] (``convert_to_fp8_block(w, is_2d_block=True)``); the result has x's type.  x is quantised in
    the weight's format, in blocks of a row.  Not differentiable."""
    _check_serving("fp8_block_linear", x, w_codes, w_scales, 2)
    return _serve(x, w_codes, w_scales, None)


@L.traced("fp8_block_grouped_linear")
def fp8_block_grouped_linear(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor, offs: torch.Tensor) -> torch.Tensor:
    """The same for rows x [M, K] that lie sorted by expert: codes [E, N, K], scales [E, ceil(N / 128), ceil(K / 128)], ``offs``
    [E] the ends of the experts' rows (any number of rows each, none too).  Rows from offs[-1] on give zeros.  Nothing
    synchronises with the host."""
    _check_serving("fp8_block_grouped_linear", x, w_codes, w_scales, 3)
    if x.dim() != 2:
        raise ValueError(f"fp8_block_grouped_linear expects rows [M, K], got {tuple(x.shape)}")
    return _serve(x, w_codes, w_scales, _ends("fp8_block_grouped_linear", offs, w_codes.shape[0], x.device))


def _ends(name: str, offs: torch.Tensor, experts: int, device) -> torch.Tensor:
    if offs.dtype not in (torch.int32, torch.int64) or offs.dim() != 1 or offs.shape[0] != experts or offs.device != device:
        raise ValueError(f"{name} expects offs as int32 [{experts}] on {device}, got {tuple(offs.shape)}, {offs.dtype} on {offs.device}")
    if experts == 0:
        raise ValueError(f"{name} expects at least one expert")
    return offs.to(torch.int32).contiguous()


# ---------------------------------------------------------------------------------------------
# training
# ---------------------------------------------------------------------------------------------
def _backward_products(ctx, grad, x_t, w_other, w_scale, offs):
    """(dx, dw in the layout [experts or 1, rows of the weight that x meets ...]) - see the two functions."""
    (M, K, N), fmt = ctx.dims, ctx.fmt
    need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
    g2 = _rows(grad)
    by_row, by_col = L.fp8_block_quantize(g2, fmt, need_x, need_w, offs) if need_x or need_w else (None, None)
    dx = dw = None
    if need_x:
        dx = torch.empty(ctx.shape, dtype=grad.dtype, device=grad.device)
        L.fp8_block_gemm(by_row[0], _row_scales(by_row[1]), w_other, w_scale, dx, fmt, (M, K, N), 0 if offs is None else 1, offs)
    if need_w:
        if offs is None:
            dw = torch.empty((N, K), dtype=grad.dtype, device=grad.device)
            if M == 0:
                dw.zero_()
            else:
                L.fp8_block_gemm(by_col[0], _row_scales(by_col[1]), x_t[0], _row_scales(x_t[1]), dw, fmt, (N, K, by_col[0].shape[1]))
        else:
            dw = torch.empty((offs.numel(), K, N), dtype=grad.dtype, device=grad.device)
            L.fp8_block_gemm(x_t[0], _row_scales(x_t[1]), by_col[0], _row_scales(by_col[1]), dw, fmt, (K, N, by_col[0].shape[1]), 2, offs, M)
    return dx, dw


class FP8BlockLinearFunction(torch.autograd.Function):
    """y = x W^T, x in blocks of a row and W [N, K] in squares; dx from the gradient in blocks of a row, dW from the gradient and
    x in blocks of 128 tokens.  What is kept is codes: of x along its columns (where W requires a gradient), of W."""

    @staticmethod
    def forward(ctx, x, weight, fp8_variant: str = "e4m3"):
        weight = unwrap_weight_wrapper(weight)
        _check_format(fp8_variant)
        if not x.is_cuda or not weight.is_cuda:
            raise RuntimeError("FP8BlockLinearFunction runs on CUDA tensors only (no CPU fallback)")
        if x.dtype not in _TYPES:
            raise ValueError(f"x dtype must be float32/bfloat16, got {x.dtype}")
        if weight.dtype != x.dtype:
            raise ValueError(f"weight dtype ({weight.dtype}) must match x dtype ({x.dtype})")
        if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
            raise ValueError(f"FP8BlockLinearFunction expects x [..., K] and a weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
        if weight.device != x.device:
            raise ValueError("FP8BlockLinearFunction expects x and weight on one device")
        N, K = weight.shape
        if N % 16 != 0 or K % 16 != 0 or N == 0 or K == 0:
            raise ValueError(f"FP8BlockLinearFunction expects features in multiples of 16, got in={K}, out={N}")
        fmt = _FMT[fp8_variant]
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        x2 = _rows(x.detach())
        M = x2.shape[0]
        w_k, w_n, w_s = L.fp8_block_quantize_squares(_rows(weight.detach()).unsqueeze(0), fmt, True, need_x)
        by_row, x_t = L.fp8_block_quantize(x2, fmt, True, need_w)
        out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
        L.fp8_block_gemm(by_row[0], _row_scales(by_row[1]), w_k, _square_scales(w_s), out, fmt, (M, N, K))
        ctx.save_for_backward(*([None, None] if x_t is None else x_t), *([None, None] if w_n is None else [w_n, w_s]))
        ctx.dims, ctx.shape, ctx.fmt = (M, K, N), x.shape, fmt
        return out

    @staticmethod
    @L.once_differentiable
    def backward(ctx, grad):
        xc, xs, w_n, w_s = ctx.saved_tensors
        dx, dw = _backward_products(ctx, grad, (xc, xs), w_n, None if w_s is None else _square_scales(w_s, True), None)
        return dx, dw, None


class GroupedFP8BlockFunction(torch.autograd.Function):
    """y[m] = x[m] B[e(m)] for B [E, K, N] and rows sorted by expert, ends in ``offs``, any number of rows an expert."""

    @staticmethod
    def forward(ctx, x, B, offs, fp8_variant: str = "e4m3"):
        name = "_quantize_then_fp8_block_scaled_grouped_mm"
        B = unwrap_weight_wrapper(B)
        _check_format(fp8_variant)
        if not x.is_cuda or not B.is_cuda:
            raise RuntimeError(f"{name} runs on CUDA tensors only (no CPU fallback)")
        if x.dtype not in _TYPES:
            raise ValueError(f"A dtype must be float32/bfloat16, got {x.dtype}")
        if B.dtype != x.dtype:
            raise ValueError(f"B dtype ({B.dtype}) must match A dtype ({x.dtype})")
        if x.dim() != 2 or B.dim() != 3 or B.shape[1] != x.shape[1]:
            raise ValueError(f"{name} expects A [M, K] and B [E, K, N], got {tuple(x.shape)} and {tuple(B.shape)}")
        if B.device != x.device:
            raise ValueError(f"{name} expects A and B on one device")
        experts, K, N = B.shape
        if N % 16 != 0 or K % 16 != 0 or N == 0 or K == 0:
            raise ValueError(f"{name} expects features in multiples of 16, got in={K}, out={N}")
        offs = _ends(name, offs, experts, x.device)
        fmt = _FMT[fp8_variant]
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        x2 = _rows(x.detach())
        M = x2.shape[0]
        b = B.detach()
        if b.stride(2) == 1 or b.stride(1) != 1:      # [K, N] in memory
            w_n, w_k, w_s = L.fp8_block_quantize_squares(_packed(b), fmt, need_x, True)
            stored_t = True
        else:                                         # [N, K]
            w_k, w_n, w_s = L.fp8_block_quantize_squares(_packed(b.transpose(1, 2)), fmt, True, need_x)
            stored_t = False
        by_row, x_t = L.fp8_block_quantize(x2, fmt, True, need_w, offs)
        out = torch.empty((M, N), dtype=x.dtype, device=x.device)
        L.fp8_block_gemm(by_row[0], _row_scales(by_row[1]), w_k, _square_scales(w_s, stored_t), out, fmt, (M, N, K), 1, offs)
        ctx.save_for_backward(offs, *([None, None] if x_t is None else x_t), *([None, None] if w_n is None else [w_n, w_s]))
        ctx.dims, ctx.shape, ctx.fmt, ctx.stored_t = (M, K, N), x.shape, fmt, stored_t
        return out

    @staticmethod
    @L.once_differentiable
    def backward(ctx, grad):
        offs, xc, xs, w_n, w_s = ctx.saved_tensors
        dx, dw = _backward_products(ctx, grad, (xc, xs), w_n, None if w_s is None else _square_scales(w_s, not ctx.stored_t), offs)
        return dx, dw, None, None


@L.on_device_of
def _linear(a, b, fp8_variant):
    return FP8BlockLinearFunction.apply(a, b, fp8_variant)


@L.traced("fp8_block_linear_training")
def _to_fp8_block_then_scaled_mm(a: torch.Tensor, b: torch.Tensor, fp8_variant: str = "e4m3") -> torch.Tensor:
    """a b^T of a training step: a [..., K], b [N, K] (bf16 or fp32, a wrapped weight too), differentiable in both."""
    if not a.is_cuda:
        raise RuntimeError("FP8BlockLinearFunction runs on CUDA tensors only (no CPU fallback)")
    a, b = outside_of_grad_mode(a, b)
    return _linear(a, b, fp8_variant)


@L.on_device_of
def _grouped(a, b, offs, fp8_variant):
    return GroupedFP8BlockFunction.apply(a, b, offs, fp8_variant)
