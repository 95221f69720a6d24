"""FP8 with one fp32 scale for each block of 128 on the GPU: quantizers bit for bit, products and gradients against 64 bits."""
import pytest
import torch

from alto_b200 import fp8_block as FB
from alto_b200 import grouped
from tests import fp8_block_helpers as H

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


def same_bits(a, b):
    a, b = a.detach().cpu().contiguous(), b.contiguous()
    return a.shape == b.shape and torch.equal(a.view(torch.uint8 if a.element_size() == 1 else torch.int32),
                                              b.view(torch.uint8 if b.element_size() == 1 else torch.int32))


# ---------------------------------------------------------------------------------------------
# quantizers
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("shape", [(1, 16), (7, 128), (128, 144), (129, 2880), (300, 272), (1024, 512)])
def test_codes_and_scales(shape, fmt, dtype):
    x = H.numbers(shape, dtype, shape[0] + shape[1])
    x[0, :16] = 0.0
    if shape[0] > 4:
        x[3] = 0.0                    # a block of zeros takes the least scale
        x[4] = x[4] * 1e-30           # and so does one of tiny numbers
    for axis in (-1, -2):
        codes, scales = FB.convert_to_fp8_block(x.cuda(), fp8_format=fmt, axis=axis)
        c, s, v = H.quantize(x, fmt, axis)
        assert same_bits(scales, s) and same_bits(codes, c)
        for out in DTYPES:
            back = FB.convert_from_fp8_block(codes, scales, out, axis=axis)
            assert torch.equal(back.cpu(), (c.float() * s.repeat_interleave(128, 1 if axis == -1 else 0)[:shape[0], :shape[1]]).to(out))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("shape", [(16, 16), (128, 128), (144, 2880), (272, 400)])
def test_squares(shape, fmt, dtype):
    w = torch.stack([H.numbers(shape, dtype, i, 0.02) for i in range(3)])
    for axis in (-1, -2):
        codes, scales = FB.convert_to_fp8_block(w.cuda(), fp8_format=fmt, axis=axis, is_2d_block=True)
        for i in range(3):
            c, s, v = H.quantize(w[i], fmt, None)
            assert same_bits(scales[i], s) and same_bits(codes[i], c)
        back = FB.convert_from_fp8_block(codes, scales, axis=axis, is_2d_block=True).cpu()
        assert torch.equal(back[2].double(), v.float().double())


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_infinities_and_nan(fmt):
    for dtype in DTYPES:
        x = H.numbers((200, 272), dtype, 5)
        x[5, 7], x[6, 140], x[199, 271], x[130, 3] = float("inf"), float("-inf"), float("nan"), 3e38
        for axis in (-1, -2):
            codes, scales = FB.convert_to_fp8_block(x.cuda(), fp8_format=fmt, axis=axis)
            c, s, v = H.quantize(x, fmt, axis)
            # (the sign of a NaN is nobody's)
            assert torch.equal(torch.isnan(scales.cpu()), torch.isnan(s)) and torch.equal(scales.cpu().nan_to_num(7.0), s.nan_to_num(7.0))
            got = codes.cpu().float()
            assert torch.equal(torch.isnan(got), torch.isnan(c.float())) and torch.equal(got.nan_to_num(7.0), c.float().nan_to_num(7.0))


def test_strides_and_leading_dimensions():
    x = H.numbers((3, 40, 400), torch.bfloat16, 1)
    wide = x.cuda()[:, :, 16:288]                   # rows of a wider buffer
    odd = x.cuda()[:, :, 3:275]                     # off 16 bytes
    for view, plain in ((wide, x[:, :, 16:288]), (odd, x[:, :, 3:275]), (x.cuda()[:, ::2, :272], x[:, ::2, :272]),
                        (x.cuda()[:1, :1, :272].expand(3, 40, 272), x[:1, :1, :272].expand(3, 40, 272))):
        for axis in (-1, -2):
            codes, scales = FB.convert_to_fp8_block(view, axis=axis)
            for i in range(3):
                c, s, _ = H.quantize(plain[i], "e4m3", axis)
                assert same_bits(scales[i], s) and same_bits(codes[i], c)
            back = FB.convert_from_fp8_block(codes, scales, axis=axis)
            assert back.shape == view.shape and bool(torch.isfinite(back).all())


# ---------------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 16, 16), (3, 144, 2880), (33, 272, 128), (128, 256, 512), (257, 512, 144), (300, 400, 1040), (515, 768, 4096)])
def test_product(m, n, k, out, fmt):
    a, b = H.numbers((m, k), torch.float32, m + k), H.numbers((n, k), torch.float32, n, 0.1)
    ca, sa, va = H.quantize(a, fmt, -1)
    for dim in (None, -1):
        cb, sb, vb = H.quantize(b, fmt, dim)
        got = FB.blockwise_fp8_gemm(ca.cuda(), sa.cuda(), cb.cuda(), sb.cuda(), output_dtype=out)
        H.assert_within(got, *H.product_bound(va, vb, out), f"{dim}")
    ca, sa, va = H.quantize(a, fmt, None)
    cb, sb, vb = H.quantize(b, fmt, None)
    got = FB.blockwise_fp8_gemm(ca.cuda(), sa.cuda().t().contiguous().t(), cb.cuda(), sb.cuda(), output_dtype=out)
    H.assert_within(got, *H.product_bound(va, vb, out), "squares on both sides")


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m,n,k", [(300, 512, 2880), (513, 272, 1040), (1100, 1040, 400), (7, 144, 2880), (200, 2064, 272)])
def test_product_with_scales_of_rows_in_either_order(m, n, k, out, fmt):
    # as a quantizer writes them (a view of [blocks, rows]) and without gaps, which go through other kernels where rows are many
    a, b = H.numbers((m, k), torch.float32, m + k), H.numbers((n, k), torch.float32, n, 0.1)
    (ca, sa, va), (cb, sb, vb) = H.quantize(a, fmt, -1), H.quantize(b, fmt, -1)
    exact, bound = H.product_bound(va, vb, out)
    ca, sa, cb, sb = (t.cuda() for t in (ca, sa, cb, sb))
    for left in (sa, sa.t().contiguous().t()):
        for right in (sb, sb.t().contiguous().t()):
            H.assert_within(FB.blockwise_fp8_gemm(ca, left, cb, right, output_dtype=out), exact, bound)
    qb, ws = FB.convert_to_fp8_block(b.cuda(), fp8_format=fmt)
    assert ws.stride() == (1, n) and torch.equal(ws, sb)
    H.assert_within(FB.blockwise_fp8_gemm(ca, sa, qb, ws, output_dtype=out), exact, bound)


@pytest.mark.parametrize("m,n,k", [(600, 1040, 128), (600, 1040, 96), (520, 2064, 1040), (40, 256, 272)])
def test_every_order_of_the_scales_gives_the_same_bits(m, n, k):
    a, b = H.numbers((m, k), torch.float32, m + k), H.numbers((n, k), torch.float32, n, 0.1)
    (ca, sa, va), (cb, sb, vb) = H.quantize(a, "e4m3", -1), H.quantize(b, "e4m3", -1)
    ca, sa, cb, sb = (t.cuda() for t in (ca, sa, cb, sb))
    best = sb.t().contiguous().t()
    want = FB.blockwise_fp8_gemm(ca, sa, cb, best, output_dtype=torch.float32)
    H.assert_within(want, *H.product_bound(va, vb, torch.float32))
    chunks = sb.shape[1]
    gaps = torch.zeros(chunks, n + 3, device="cuda")[:, :n].t()           # neighbours along the rows, blocks an odd number apart
    shifted = torch.zeros(chunks * n + 1, device="cuda")[1:].view(chunks, n).t()
    spread = torch.zeros(n, 2 * chunks, device="cuda")[:, ::2]
    for s in (sb, gaps, shifted, spread):
        s.copy_(sb)
        got = FB.blockwise_fp8_gemm(ca, sa, cb, s, output_dtype=torch.float32)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 8, 9, 16, 17, 40, 200])
def test_serving(m, dtype):
    for n, k, fmt in ((144, 2880, "e4m3"), (512, 256, "e5m2"), (4096, 128, "e4m3")):
        x, w = H.numbers((m, k), dtype, m), H.numbers((n, k), torch.float32, n, 0.05)
        c, s = FB.convert_to_fp8_block(w.cuda(), fp8_format=fmt, is_2d_block=True)
        got = FB.fp8_block_linear(x.cuda(), c, s)
        assert got.dtype == dtype
        H.assert_within(got, *H.product_bound(H.quantize(x, fmt, -1)[2], H.quantize(w, fmt, None)[2], dtype), f"{n} {k}")


COUNTS = [[5], [0, 3, 0, 1], [128, 128, 256], [1, 127, 129, 0, 300, 2], [0, 0, 0], [700, 0, 5], [3] * 40]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", COUNTS, ids=str)
def test_serving_by_expert(counts, dtype):
    e, n, k, spare = len(counts), 272, 400, 7
    rows = sum(counts) + spare
    x, w = H.numbers((rows, k), dtype, rows), torch.stack([H.numbers((n, k), torch.float32, i, 0.05) for i in range(e)])
    c, s = FB.convert_to_fp8_block(w.cuda(), is_2d_block=True)
    got = FB.fp8_block_grouped_linear(x.cuda(), c, s, H.runs(counts).cuda())
    at = 0
    for i, m in enumerate(counts):
        if m:
            H.assert_within(got[at:at + m], *H.product_bound(H.quantize(x[at:at + m], "e4m3", -1)[2], H.quantize(w[i], "e4m3", None)[2], dtype), f"expert {i}")
        at += m
    assert not bool(got[at:].any())


# ---------------------------------------------------------------------------------------------
# training
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("m,n,k", [(1, 16, 32), (37, 144, 208), (200, 400, 272), (384, 256, 512), (1000, 272, 2880)])
def test_linear_and_gradients(m, n, k, fmt, dtype):
    x, w, dy = H.numbers((m, k), dtype, 1), H.numbers((n, k), dtype, 2, 0.05), H.numbers((m, n), dtype, 3, 1e-3)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = FB._to_fp8_block_then_scaled_mm(xg, wg, fp8_variant=fmt)
    dx, dw = torch.autograd.grad((y,), (xg, wg), (dy.cuda(),))
    wv = H.quantize(w, fmt, None)[2]
    H.assert_within(y, *H.product_bound(H.quantize(x, fmt, -1)[2], wv, dtype), "y")
    H.assert_within(dx, *H.product_bound(H.quantize(dy, fmt, -1)[2], wv.T, dtype), "dx")
    H.assert_within(dw, *H.product_bound(H.quantize(dy, fmt, -2)[2].T, H.quantize(x, fmt, -2)[2].T, dtype), "dw")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("counts", COUNTS, ids=str)
def test_grouped_and_gradients(counts, stored, dtype):
    e, n, k, spare, fmt = len(counts), 272, 400, 5, "e4m3"
    rows = sum(counts) + spare
    x, dy = H.numbers((rows, k), dtype, 1), H.numbers((rows, n), dtype, 3, 1e-3)
    w = torch.stack([H.numbers((k, n), dtype, i, 0.05) for i in range(e)])
    xg = x.cuda().requires_grad_(True)
    wg = w.cuda() if stored == "kn" else w.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    wg.requires_grad_(True)
    y = grouped._quantize_then_fp8_block_scaled_grouped_mm(xg, wg, offs=H.runs(counts).cuda(), fp8_variant=fmt)
    dx, dw = torch.autograd.grad((y,), (xg, wg), (dy.cuda(),))
    assert dw.shape == w.shape
    at = 0
    for i, m in enumerate(counts):
        if m:
            rs, wv = slice(at, at + m), H.quantize(w[i], fmt, None)[2]
            H.assert_within(y[rs], *H.product_bound(H.quantize(x[rs], fmt, -1)[2], wv.T, dtype), f"y of {i}")
            H.assert_within(dx[rs], *H.product_bound(H.quantize(dy[rs], fmt, -1)[2], wv, dtype), f"dx of {i}")
            H.assert_within(dw[i], *H.product_bound(H.quantize(x[rs], fmt, -2)[2].T, H.quantize(dy[rs], fmt, -2)[2].T, dtype), f"dw of {i}")
        else:
            assert not bool(dw[i].any())
        at += m
    assert not bool(y[at:].any()) and not bool(dx[at:].any())
