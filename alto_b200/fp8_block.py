"""FP8 with one fp32 scale for each block of 128: quantizers, the product, and linears dense and grouped by expert, on B200.

    convert_to_fp8_block / convert_from_fp8_block      codes and scales along an axis, or of squares of 128 x 128
    blockwise_fp8_gemm(a, a_s, b, b_s)                 a b^T of two quantised operands
    _to_fp8_block_then_scaled_mm                       a training step's linear (x in blocks of a row, weights in squares; the
                                                       weight gradient in blocks of tokens); its autograd function is C++
    fp8_block_linear / fp8_block_grouped_linear        serving: weights that are there as codes and scales, from one token up

A block's scale is max(|largest|, 1e-12) / top (top: 448 for E4M3, 57344 for E5M2) and its codes are the quotients by it, to
nearest; a last block is as short as the dimension.  The products of a block of 128 are summed by the tensor cores and added
up in fp32 with both scales.  Features (in and out) are multiples of 16, tokens any number.  The grouped training form is
``grouped._quantize_then_fp8_block_scaled_grouped_mm``.

The reference has this format in a part that its recipes do not reach (alto/kernels/blockwise_fp8/blockwise_linear.py:161);
recipes name it here as the schemes "fp8_block_e4m3" and "fp8_block_e5m2" (``dispatch.TrainingOpConfig``, ``lpt.LowPrecisionTrainingModifier``)."""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib as L
from .nvfp4 import unwrap_weight_wrapper

__all__ = ["convert_to_fp8_block", "convert_from_fp8_block", "blockwise_fp8_gemm", "fp8_block_linear",
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
    x3 = x.reshape(math.prod(lead), M, N)
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


def _many(M: int, N: int) -> bool:
    """Whether a product is not for the kernel of few rows, which takes scales in any order (16 rows, or two rounds of tiles of 32 x 32
    on 148 SMs)."""
    return M > 16 and -(-M // 32) * -(-N // 32) > 296


@L.traced("blockwise_fp8_gemm")
def blockwise_fp8_gemm(a: torch.Tensor, a_s: torch.Tensor, b: torch.Tensor, b_s: torch.Tensor,
                       output_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a b^T for codes a [M, K] and b [N, K] of one format with fp32 scales [M or ceil(M / 128), ceil(K / 128)] and
    [N or ceil(N / 128), ceil(K / 128)]; N and K multiples of 16.  Scales lie in any order; those of b's rows that are not neighbours along
    the rows, as ``convert_to_fp8_block`` returns them for a matrix, are copied into that order where rows are many."""
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
    sides, kept = [], None
    for name, s, rows in (("a_s", a_s, M), ("b_s", b_s, N)):
        if s.dtype != torch.float32 or s.dim() != 2 or s.shape[1] != _blocks(K) or s.shape[0] not in (rows, _blocks(rows)):
            raise ValueError(f"blockwise_fp8_gemm expects fp32 scales {name} [{rows} or {_blocks(rows)}, {_blocks(K)}], got "
                             f"{tuple(s.shape)}, {s.dtype}")
        chunk = s.stride(1) if s.shape[1] > 1 else rows
        if name == "b_s" and s.shape[0] == rows and _many(M, N) and (s.stride(0) != 1 or chunk % 4 != 0 or s.data_ptr() % 16 != 0):
            s = kept = s.detach().t().clone(memory_format=torch.contiguous_format).t()
            chunk = rows
        sides.append(L.Fp8BlockScale(s.data_ptr(), s.stride(0), chunk, 0, 0 if s.shape[0] == rows else 7, 7))
    if any(t.device != a.device for t in (a_s, b, b_s)):
        raise ValueError("blockwise_fp8_gemm expects all tensors on one device")
    out = torch.empty((M, N), dtype=output_dtype, device=a.device)
    a8, b8 = _packed(a.detach()).view(torch.uint8), _packed(b.detach()).view(torch.uint8)
    L.fp8_block_gemm(a8, sides[0], b8, sides[1], out, _FMT_OF_DTYPE[a.dtype], (M, N, K))
    return out


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
    if torch.is_grad_enabled() and (x.requires_grad or w_scales.requires_grad):
        raise RuntimeError(f"{name} has no gradient: codes of weights serve evaluation")
    if L.forward_mode() and any(forward_ad.unpack_dual(t).tangent is not None for t in (x, w_scales)):
        raise RuntimeError(f"{name} has no forward-mode derivative")


@L.traced("fp8_block_linear")
def fp8_block_linear(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor) -> torch.Tensor:
    """x W^T for x [..., K] (bf16 or fp32) and a weight that is there as codes [N, K] and fp32 scales of its squares
    [ceil(N / 128), ceil(K / 128)] (``convert_to_fp8_block(w, is_2d_block=True)``); the result has x's type.  x is quantised in
    the weight's format, in blocks of a row.  Not differentiable."""
    host = L._autograd_module or L.autograd()
    if not L.forward_mode():
        y = host.fp8_try_serve(x, w_codes, w_scales, None)
        if y is not None:
            return y
    _check_serving("fp8_block_linear", x, w_codes, w_scales, 2)
    return host.fp8_serve(x, w_codes, w_scales, None, _FMT_OF_DTYPE[w_codes.dtype])


@L.traced("fp8_block_grouped_linear")
def fp8_block_grouped_linear(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor, offs: torch.Tensor) -> torch.Tensor:
    """The same for rows x [M, K] that lie sorted by expert: codes [E, N, K], scales [E, ceil(N / 128), ceil(K / 128)], ``offs``
    [E] the ends of the experts' rows (any number of rows each, none too).  Rows from offs[-1] on give zeros.  Nothing
    synchronises with the host."""
    host = L._autograd_module or L.autograd()
    if offs is not None and not L.forward_mode():
        y = host.fp8_try_serve(x, w_codes, w_scales, offs)
        if y is not None:
            return y
    _check_serving("fp8_block_grouped_linear", x, w_codes, w_scales, 3)
    if x.dim() != 2:
        raise ValueError(f"fp8_block_grouped_linear expects rows [M, K], got {tuple(x.shape)}")
    offs = _ends("fp8_block_grouped_linear", offs, w_codes.shape[0], x.device)
    return host.fp8_serve(x, w_codes, w_scales, offs, _FMT_OF_DTYPE[w_codes.dtype])


def _ends(name: str, offs: torch.Tensor, experts: int, device) -> torch.Tensor:
    if not isinstance(offs, torch.Tensor):
        raise ValueError(f"{name} expects offs as int32 [{experts}] on {device}, got {type(offs).__name__}")
    if offs.dtype not in (torch.int32, torch.int64) or offs.dim() != 1 or offs.shape[0] != experts or offs.device != device:
        raise ValueError(f"{name} expects offs as int32 [{experts}] on {device}, got {tuple(offs.shape)}, {offs.dtype} on {offs.device}")
    if experts == 0:
        raise ValueError(f"{name} expects at least one expert")
    if offs.dtype is torch.int32 and offs.is_contiguous():
        return offs
    if offs.dtype is torch.int64:      # an end past 31 bits is past the buffer, too
        offs = offs.clamp(-1, 2 ** 31 - 1)
    return offs.to(torch.int32).contiguous()


# ---------------------------------------------------------------------------------------------
# training
# ---------------------------------------------------------------------------------------------
def _plain(weight: torch.Tensor) -> torch.Tensor:
    return weight if type(weight) is torch.Tensor or type(weight) is torch.nn.Parameter else unwrap_weight_wrapper(weight)


def _check_training(name: str, x: torch.Tensor, w: torch.Tensor, dims: int, fp8_variant: str) -> None:
    _check_format(fp8_variant)
    if not x.is_cuda or not w.is_cuda:
        raise RuntimeError(f"{name} runs on CUDA tensors only (no CPU fallback)")
    if x.dtype not in _TYPES:
        raise ValueError(f"A dtype must be float32/bfloat16, got {x.dtype}")
    if w.dtype != x.dtype:
        raise ValueError(f"weight dtype ({w.dtype}) must match the activations' ({x.dtype})")
    if w.dim() != dims or x.dim() < 1 or (dims == 3 and x.dim() != 2) or x.shape[-1] != w.shape[1]:
        raise ValueError(f"{name} expects " + ("A [..., K] and B [N, K]" if dims == 2 else "A [M, K] and B [E, K, N]") +
                         f", got {tuple(x.shape)} and {tuple(w.shape)}")
    if w.device != x.device:
        raise ValueError(f"{name} expects all tensors on one device")
    if any(n % 16 != 0 or n == 0 for n in w.shape[-2:]):
        raise ValueError(f"{name} expects features in multiples of 16, got {tuple(w.shape[-2:])}")


@L.traced("fp8_block_linear_training")
def _to_fp8_block_then_scaled_mm(a: torch.Tensor, b: torch.Tensor, fp8_variant: str = "e4m3") -> torch.Tensor:
    """a b^T of a training step: a [..., K], b [N, K] (bf16 or fp32, a wrapped weight too), differentiable in both.  a is quantised
    in blocks of a row and b in squares; the gradient of a takes the upstream one in blocks of a row, that of b both in blocks
    of 128 tokens.  What is kept is codes: of a along its columns (where b requires a gradient) and of b."""
    host = L._autograd_module or L.autograd()
    if fp8_variant in _FMT:
        y = host.fp8_try_linear(a, b, None, _FMT[fp8_variant])
        if y is not None:
            return y
    w = _plain(b)
    _check_training("_to_fp8_block_then_scaled_mm", a, w, 2, fp8_variant)
    return host.fp8_linear(a, b, w, None, _FMT[fp8_variant])


def _grouped(a: torch.Tensor, b: torch.Tensor, offs: torch.Tensor, fp8_variant: str) -> torch.Tensor:
    name = "_quantize_then_fp8_block_scaled_grouped_mm"
    host = L._autograd_module or L.autograd()
    if offs is not None and fp8_variant in _FMT:
        y = host.fp8_try_linear(a, b, offs, _FMT[fp8_variant])
        if y is not None:
            return y
    w = _plain(b)
    _check_training(name, a, w, 3, fp8_variant)
    return host.fp8_linear(a, b, w, _ends(name, offs, w.shape[0], a.device), _FMT[fp8_variant])
