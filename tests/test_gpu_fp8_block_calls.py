"""The FP8 block operators as they are called: wrapped weights, recipes, parts of the gradients, views, streams, captured graphs, bad ends,
numbers that are not finite, long buffers, many experts, refusals, and a step of a model with all of them."""
import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

import alto_b200.dispatch as D
from alto_b200 import fp8_block as FB
from alto_b200 import grad_clip, grouped
from alto_b200.lpt import LowPrecisionTrainingModifier
from tests import fp8_block_helpers as H

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
CONFIG = D.TrainingOpConfig(precision="fp8_block_e4m3", use_2dblock_x=False, use_2dblock_w=True, use_hadamard=False, use_sr_grad=False, use_dge=False)


def wrapped(w, **kw):
    return nn.Parameter(D.FP8BlockTrainingWeightWrapperTensor(w, CONFIG), **kw)


# ---------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------
def test_refusals_of_quantizers_and_products():
    x = torch.zeros(32, 64, device="cuda", dtype=BF)
    for bad in (dict(fp8_format="e3m4"), dict(block_size=64), dict(axis=0 - 3), dict(axis=2)):
        with pytest.raises(ValueError):
            FB.convert_to_fp8_block(x, **bad)
    for t, kw in ((x[:, :40], {}), (x[0], {}), (x[:, :0], {}), (x[:20], dict(is_2d_block=True)), (x[:0], dict(is_2d_block=True))):
        with pytest.raises(ValueError):
            FB.convert_to_fp8_block(t, **kw)
    with pytest.raises(TypeError):
        FB.convert_to_fp8_block(x.half())
    codes, scales = FB.convert_to_fp8_block(x)
    for c, s, kw in ((codes, scales[:31], {}), (codes, scales.double(), {}), (codes.view(torch.uint8), scales, {}), (codes, scales, dict(block_size=32)),
                     (codes, scales, dict(axis=-2)), (codes, scales, dict(is_2d_block=True)), (codes, scales.cpu(), {}), (codes[:, :4], scales, {})):
        with pytest.raises((ValueError, RuntimeError)):
            FB.convert_from_fp8_block(c, s, **kw)
    with pytest.raises(TypeError):
        FB.convert_from_fp8_block(codes, scales, torch.float16)
    other = codes.float().to(torch.float8_e5m2)
    for a, sa, b, sb in ((codes, scales, other, scales), (codes[:, :24], scales, codes[:, :24], scales), (codes, scales, codes[:24], scales[:24]),
                         (codes, scales[:3], codes, scales), (codes, scales, codes, scales.half()), (codes, scales, codes[:, :48], scales),
                         (codes[0], scales, codes, scales), (codes, scales, codes[:0], scales[:0]), (x, scales, x, scales)):
        with pytest.raises(ValueError):
            FB.blockwise_fp8_gemm(a, sa, b, sb)
    with pytest.raises(TypeError):
        FB.blockwise_fp8_gemm(codes, scales, codes, scales, torch.float16)


def test_refusals_of_linears():
    x, w = torch.zeros(32, 64, device="cuda", dtype=BF), torch.zeros(48, 64, device="cuda", dtype=BF)
    codes, scales = FB.convert_to_fp8_block(w, is_2d_block=True)
    offs = torch.tensor([32], device="cuda", dtype=torch.int32)
    for a, c, s, kind in ((x.half(), codes, scales, TypeError), (x, codes.view(torch.uint8), scales, ValueError), (x[:, :48], codes, scales, ValueError),
                          (x, codes, scales[0], ValueError), (x, codes, scales.half(), ValueError), (x, codes[None], scales, ValueError),
                          (x, codes[:40], scales, ValueError), (x, codes[:0], scales[:0], ValueError), (x[:, :40], codes[:, :40], scales, ValueError),
                          (x, codes, scales.cpu(), RuntimeError), (x.clone().requires_grad_(True), codes, scales, RuntimeError)):
        with pytest.raises(kind):
            FB.fp8_block_linear(a, c, s)
    for a, o in ((x[None], offs), (x, offs.float()), (x, offs.cpu()), (x, offs[None]), (x, torch.cat([offs, offs]))):
        with pytest.raises(ValueError):
            FB.fp8_block_grouped_linear(a, codes[None], scales[None], o)
    for a, b, kw in ((x, w.float(), {}), (x.half(), w.half(), {}), (x[:, :48], w, {}), (x, w[:40], {}), (x, w[:0], {}), (x, w[None], {}),
                     (x, w, dict(fp8_variant="e3m4"))):
        with pytest.raises(ValueError):
            FB._to_fp8_block_then_scaled_mm(a, b, **kw)
    with pytest.raises(RuntimeError):
        FB._to_fp8_block_then_scaled_mm(x, w.cpu())
    b = w.t()[None]
    for a, bb, o in ((x[None], b, offs), (x, b[0], offs), (x, b, offs.float()), (x, b, offs[:0]), (x, b[:, :, :40], offs), (x, b.float(), offs)):
        with pytest.raises(ValueError):
            grouped._quantize_then_fp8_block_scaled_grouped_mm(a, bb, offs=o)


@pytest.mark.parametrize("m", [4, 40])
def test_a_gradient_of_the_scales_is_not_dropped(m):
    x, w = torch.randn(m, 64, device="cuda", dtype=BF), torch.randn(48, 64, device="cuda", dtype=BF)
    codes, scales = FB.convert_to_fp8_block(w, is_2d_block=True)
    offs = torch.tensor([m], device="cuda", dtype=torch.int32)
    calls = (lambda s: FB.fp8_block_linear(x, codes, s), lambda s: FB.fp8_block_grouped_linear(x, codes[None], s[None], offs))
    wants = [call(scales) for call in calls]
    scales.requires_grad_(True)
    for call, want in zip(calls, wants):
        with pytest.raises(RuntimeError, match="no gradient"):
            call(scales)
        with torch.no_grad():
            assert torch.equal(call(scales), want)


def test_a_tangent_is_not_dropped():
    x, w = torch.randn(32, 64, device="cuda", dtype=BF), torch.randn(48, 64, device="cuda", dtype=BF)
    codes, scales = FB.convert_to_fp8_block(w, is_2d_block=True)
    offs = torch.tensor([32], device="cuda", dtype=torch.int32)
    want = FB._to_fp8_block_then_scaled_mm(x, w), FB.fp8_block_linear(x, codes, scales)
    for grad in (True, False):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            d, dw = forward_ad.make_dual(x, torch.randn_like(x)), forward_ad.make_dual(w, torch.randn_like(w))
            for call in (lambda: FB._to_fp8_block_then_scaled_mm(d, w), lambda: FB._to_fp8_block_then_scaled_mm(x, dw),
                         lambda: grouped._quantize_then_fp8_block_scaled_grouped_mm(d, w.t()[None], offs=offs),
                         lambda: FB.fp8_block_linear(d, codes, scales), lambda: FB.fp8_block_grouped_linear(d, codes[None], scales[None], offs)):
                with pytest.raises(RuntimeError):
                    call()
            assert torch.equal(FB._to_fp8_block_then_scaled_mm(x, w), want[0]) and torch.equal(FB.fp8_block_linear(x, codes, scales), want[1])


def test_a_second_derivative_is_refused():
    x, w = torch.randn(32, 64, device="cuda").requires_grad_(True), torch.randn(48, 64, device="cuda").requires_grad_(True)
    dy = torch.randn(32, 48, device="cuda").requires_grad_(True)
    dx, dw = torch.autograd.grad(FB._to_fp8_block_then_scaled_mm(x, w), (x, w), dy, create_graph=True)
    for t in (dx, dw):
        with pytest.raises(RuntimeError):
            t.sum().backward(retain_graph=True)


# ---------------------------------------------------------------------------------------------
# gradients
# ---------------------------------------------------------------------------------------------
def whole(shape, seed):
    """Whole numbers of at most 8 with a 448 in every block of a row, of a column and in every square: scale one, every code exact."""
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(-8, 9, shape, generator=g).float()
    rows, cols = shape
    for r in range(rows):
        t[r, (r % 128)::128] = 448.0
    for c in range(cols):
        t[(c % 128)::128, c] = 448.0
    return t


@pytest.mark.parametrize("where", ["dense", "grouped"])
def test_gradients_against_differences(where):
    m, n, k = 256, 128, 256
    x, w, c = whole((m, k), 1).cuda(), whole((n, k), 2).cuda(), whole((m, n), 3).cuda()
    offs = torch.tensor([128, 256], device="cuda", dtype=torch.int32)

    def out(a, b):
        if where == "dense":
            return FB._to_fp8_block_then_scaled_mm(a, b)
        return grouped._quantize_then_fp8_block_scaled_grouped_mm(a, torch.stack([b.t(), b.t()]), offs=offs)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(out(xl, wl), (xl, wl), c)
    g = torch.Generator().manual_seed(4)
    for t, grad in ((x, dx), (w, dw)):
        free = (t.abs() < 8).nonzero().cpu()
        for i in torch.randint(0, len(free), (8,), generator=g).tolist():
            r, q = free[i].tolist()
            up, down = t.clone(), t.clone()
            up[r, q] += 1.0           # still a code
            down[r, q] -= 1.0
            pair = (out(up, w), out(down, w)) if t is x else (out(x, up), out(x, down))
            # products of whole numbers, sums below 2^24: exact in fp32, so is the slope of a linear function
            slope = float(((pair[0].double() - pair[1].double()) * c.double()).sum() / 2)
            assert float(grad[r, q]) == slope


@pytest.mark.parametrize("part", ["x", "w"])
def test_one_gradient_alone(part):
    x, w, dy = (H.numbers(s, BF, i).cuda() for i, s in enumerate(((300, 144), (272, 144), (300, 272))))
    both = torch.autograd.grad(FB._to_fp8_block_then_scaled_mm(x.clone().requires_grad_(True), leaf := w.clone().requires_grad_(True)), leaf, dy)
    xl, wl = x.clone().requires_grad_(part == "x"), w.clone().requires_grad_(part == "w")
    y = FB._to_fp8_block_then_scaled_mm(xl, wl)
    y.backward(dy)
    assert (xl.grad is None) == (part == "w") and (wl.grad is None) == (part == "x")
    if part == "w":
        assert torch.equal(wl.grad, both[0])
    with torch.no_grad():
        z = FB._to_fp8_block_then_scaled_mm(xl, wl)
    assert not z.requires_grad and torch.equal(z, y)
    with torch.inference_mode():
        assert torch.equal(FB._to_fp8_block_then_scaled_mm(xl, wl), y)
        c, s = FB.convert_to_fp8_block(w, is_2d_block=True)
        served = FB.fp8_block_linear(x, c, s)
    H.assert_within(served, *H.product_bound(H.quantize(x.cpu(), "e4m3", -1)[2], H.quantize(w.cpu(), "e4m3", None)[2], BF))


def test_one_token_without_a_dimension_for_it():
    x, w, dy = H.numbers((272,), BF, 1).cuda().requires_grad_(True), H.numbers((144, 272), BF, 2).cuda().requires_grad_(True), H.numbers((144,), BF, 3).cuda()
    y = FB._to_fp8_block_then_scaled_mm(x, w)
    got = (y, *torch.autograd.grad(y, (x, w), dy))
    z = FB._to_fp8_block_then_scaled_mm(x[None], w)
    want = (z, *torch.autograd.grad(z, (x, w), dy[None]))
    assert y.shape == (144,) and all(torch.equal(a, b.view(a.shape)) for a, b in zip(got, want))


def test_no_rows():
    w, x = torch.randn(48, 64, device="cuda", dtype=BF).requires_grad_(True), torch.zeros(0, 64, device="cuda", dtype=BF).requires_grad_(True)
    y = FB._to_fp8_block_then_scaled_mm(x, w)
    y.sum().backward()
    assert y.shape == (0, 48) and x.grad.shape == (0, 64) and not bool(w.grad.any())
    offs = torch.zeros(3, device="cuda", dtype=torch.int32)
    b = torch.randn(3, 64, 48, device="cuda", dtype=BF).requires_grad_(True)
    y = grouped._quantize_then_fp8_block_scaled_grouped_mm(x, b, offs=offs)
    y.sum().backward()
    assert y.shape == (0, 48) and not bool(b.grad.any())
    c, s = FB.convert_to_fp8_block(w, is_2d_block=True)
    assert FB.fp8_block_linear(x.detach(), c, s).shape == (0, 48) and FB.fp8_block_linear(x.detach().view(3, 0, 64), c, s).shape == (3, 0, 48)
    assert FB.fp8_block_grouped_linear(x.detach(), c[None], s[None], offs[:1]).shape == (0, 48)
    assert FB.blockwise_fp8_gemm(c[:0], torch.zeros(0, 1, device="cuda"), c, s).shape == (0, 48)
    assert FB.convert_to_fp8_block(x)[0].shape == (0, 64) and FB.convert_to_fp8_block(x, axis=-2)[1].shape == (0, 64)


# ---------------------------------------------------------------------------------------------
# operands as they come
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
def test_views(dtype):
    x, w, dy = H.numbers((6, 50, 272), dtype, 1).cuda(), H.numbers((400, 272), dtype, 2, 0.1).cuda(), H.numbers((6, 50, 400), dtype, 3).cuda()
    wide = torch.zeros(6, 50, 300, device="cuda", dtype=dtype)
    odd = torch.zeros(6, 50, 273, device="cuda", dtype=dtype)
    wide[..., 16:288], odd[..., 1:] = x, x

    def step(a, b, g):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y = FB._to_fp8_block_then_scaled_mm(a, b)
        return (y, *torch.autograd.grad(y, (a, b), g))
    want = step(x, w, dy)
    assert want[0].shape == (6, 50, 400) and want[1].shape == x.shape
    gaps = torch.zeros(6, 50, 800, device="cuda", dtype=dtype)[..., ::2]
    gaps.copy_(dy)
    for a, b, g in ((wide[..., 16:288], w, dy), (odd[..., 1:], w, dy), (x.transpose(0, 1).contiguous().transpose(0, 1), w, dy),
                    (x, w.t().contiguous().t(), gaps), (x, torch.cat([w, w], 1)[:, :272], dy.transpose(0, 1).contiguous().transpose(0, 1))):
        assert all(torch.equal(p, q) for p, q in zip(step(a, b, g), want))
    y = FB._to_fp8_block_then_scaled_mm(a := x.clone().requires_grad_(True), w)
    y.sum().backward()                                       # a gradient of one number
    assert torch.equal(a.grad, step(x, w, torch.ones_like(dy))[1])
    codes, scales = FB.convert_to_fp8_block(w, is_2d_block=True)
    rows = FB.fp8_block_linear(x, codes, scales)
    c2, s2 = FB.convert_to_fp8_block(w, is_2d_block=True, axis=-2)       # codes that lie by columns
    s3 = torch.zeros(4, 6, device="cuda")[:, ::2]
    s3.copy_(scales)
    assert c2.stride() == (1, 400)
    for m in (300, 20, 3):
        a = x.view(300, 272)[:m]
        want = FB.fp8_block_linear(a, codes, scales)
        assert torch.equal(want, rows.view(300, 400)[:m]) or m < 300      # (fewer rows go through another kernel)
        assert torch.equal(FB.fp8_block_linear(wide[..., 16:288].reshape(300, 272)[:m], c2, s3), want)
    assert FB.fp8_block_linear(x[0, 0], codes, scales).shape == (400,)


def test_ends_of_sixty_four_bits_and_bad_ones():
    rows, e, n, k = 300, 4, 144, 272
    x, w = H.numbers((rows, k), BF, 1).cuda(), H.numbers((e * n, k), BF, 2, 0.1).cuda().view(e, n, k)
    codes, scales = FB.convert_to_fp8_block(w, is_2d_block=True)
    good = torch.tensor([10, 10, 200, 260], device="cuda", dtype=torch.int32)
    every = torch.stack([good.long(), good.long()], 1)[:, 0]

    def run(offs, m=rows):
        xl, b = x[:m].clone().requires_grad_(True), w.transpose(1, 2).clone().requires_grad_(True)
        y = grouped._quantize_then_fp8_block_scaled_grouped_mm(xl, b, offs=offs)
        return (y, *torch.autograd.grad(y, (xl, b), torch.ones_like(y)), FB.fp8_block_grouped_linear(x[:m], codes, scales, offs))
    assert all(torch.equal(a, b) for a, b in zip(run(good), run(every)))
    # out of order or out of the buffer: taken as a running maximum, cut off at the rows
    for bad, like in (([10, 5, 200, 260], [10, 10, 200, 260]), ([-7, 50, 40, 9999], [0, 50, 50, 300]), ([2 ** 31 - 1] * 4, [300] * 4),
                      ([-2 ** 31] * 4, [0] * 4)):
        a, b = (run(torch.tensor(o, device="cuda", dtype=torch.int32)) for o in (bad, like))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        a, b = (run(torch.tensor(o, device="cuda", dtype=torch.int32).clamp(max=40 if o is like else 2 ** 31 - 1), 40) for o in (bad, like))
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_ends_past_thirty_one_bits_and_none():
    x, w = H.numbers((40, 272), BF, 1).cuda(), H.numbers((2 * 144, 272), BF, 2, 0.1).cuda().view(2, 144, 272)
    codes, scales = FB.convert_to_fp8_block(w, is_2d_block=True)
    for ends, like in (([2 ** 32 + 5, 2 ** 40], [40, 40]), ([7, 2 ** 33], [7, 40]), ([-2 ** 40, 2 ** 32], [0, 40])):
        a, b = torch.tensor(ends, device="cuda"), torch.tensor(like, device="cuda", dtype=torch.int32)
        assert torch.equal(FB.fp8_block_grouped_linear(x, codes, scales, a), FB.fp8_block_grouped_linear(x, codes, scales, b))
        assert torch.equal(grouped._quantize_then_fp8_block_scaled_grouped_mm(x, w.transpose(1, 2), offs=a),
                           grouped._quantize_then_fp8_block_scaled_grouped_mm(x, w.transpose(1, 2), offs=b))
    for bad in (None, [7, 40]):                 # (nor is a matrix taken for the experts' then)
        for c, s in ((codes, scales), (codes[0], scales[0])):
            with pytest.raises((ValueError, TypeError)):
                FB.fp8_block_grouped_linear(x, c, s, bad)
        for b in (w.transpose(1, 2), w[0], w[0].t()):
            with pytest.raises((ValueError, TypeError)):
                grouped._quantize_then_fp8_block_scaled_grouped_mm(x, b, offs=bad)


def in_order(ends, rows):
    """The running maximum of ends that are cut off at the rows."""
    return torch.cummax(ends.clamp(0, rows), 0)[0].to(torch.int32)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,e", [(1, 2), (5, 3), (8, 4), (8, 40), (20, 4), (24, 40), (90, 3), (8, 1500), (20, 1500), (300, 1500)])
def test_bad_ends_in_every_product(m, e, dtype):
    # up to eight rows, few an expert, many an expert, more experts than the lists hold
    n, k = 48, 272
    x, w = H.numbers((m, k), dtype, 1).cuda(), H.numbers((e * n, k), dtype, 2, 0.1).cuda().view(e, n, k)
    dy = H.numbers((m, n), dtype, 3).cuda()
    codes, scales = FB.convert_to_fp8_block(w, is_2d_block=True)

    def run(offs):
        xl, b = x.clone().requires_grad_(True), w.transpose(1, 2).clone().requires_grad_(True)
        y = grouped._quantize_then_fp8_block_scaled_grouped_mm(xl, b, offs=offs)
        return (FB.fp8_block_grouped_linear(x, codes, scales, offs), y, *torch.autograd.grad(y, (xl, b), dy))
    g = torch.Generator().manual_seed(m * e)
    lists = [torch.randint(-2, m + 3, (e,), generator=g) for _ in range(4)]
    lists += [torch.full((e,), m), torch.arange(e, 0, -1) * m // e, torch.cat([torch.tensor([m]), torch.zeros(e - 1, dtype=torch.long)])]
    for ends in lists:
        want = run(in_order(ends, m).cuda())
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(run(ends.to(torch.int32).cuda()), want))


@pytest.mark.parametrize("ends", [[5, 3, 8], [8, 3, 1], [6, 2, 8], [3, -4, 2], [99, 0, 1]], ids=str)
def test_bad_ends_of_up_to_eight_rows_against_the_formula(ends):
    m, n, k = 8, 144, 400
    x, w = H.numbers((m, k), F32, 1), H.numbers((3 * n, k), F32, 2, 0.1).view(3, n, k)
    codes, scales = FB.convert_to_fp8_block(w.cuda(), is_2d_block=True)
    got = FB.fp8_block_grouped_linear(x.cuda(), codes, scales, torch.tensor(ends, device="cuda", dtype=torch.int32))
    a, at = H.quantize(x, "e4m3", -1)[2], 0
    for e, end in enumerate(in_order(torch.tensor(ends), m).tolist()):
        exact, bound = H.product_bound(a[at:end], H.quantize(w[e], "e4m3", None)[2], F32)
        H.assert_within(got[at:end], exact, bound, f"expert {e}")
        at = end
    assert not bool(got[at:].any())


@pytest.mark.parametrize("m", [4, 24, 300])
def test_numbers_that_are_not_finite_stay_in_their_blocks(m):
    n, k = 272, 400
    x, w = H.numbers((m, k), BF, 1), H.numbers((n, k), BF, 2, 0.1)
    codes, scales = FB.convert_to_fp8_block(w.cuda(), is_2d_block=True)
    clean = FB.fp8_block_linear(x.cuda(), codes, scales)
    bad = x.clone()
    bad[1, 7], bad[2, 390] = float("nan"), float("inf")
    got = FB.fp8_block_linear(bad.cuda(), codes, scales)
    keep = [r for r in range(m) if r not in (1, 2)]
    assert torch.equal(got[keep], clean[keep]) and not bool(torch.isfinite(got[[1, 2]]).any())
    s = scales.clone()
    s[1, 1] = float("nan")                                   # rows 128 to 255 of the weight
    got = FB.fp8_block_linear(x.cuda(), codes, s)
    cols = [c for c in range(n) if not 128 <= c < 256]
    assert bool(torch.isnan(got[:, 128:256]).all()) and torch.equal(got[:, cols], clean[:, cols])


def test_rows_of_zeros_and_tiny_rows():
    x = torch.zeros(40, 256, device="cuda", dtype=BF)
    x[1] = 1e-30
    w = torch.randn(64, 256, device="cuda", dtype=BF)
    y = FB._to_fp8_block_then_scaled_mm(x, w)
    assert not bool(y.any()) and bool(torch.isfinite(y).all())


@pytest.mark.parametrize("m", [2, 20, 200])
def test_more_experts_than_a_list_holds(m):
    e, n, k = 1500, 48, 144
    g = torch.Generator().manual_seed(m)
    ends = torch.sort(torch.randint(0, m + 1, (e,), generator=g))[0].to(torch.int32)
    x, w = H.numbers((m, k), F32, 1), H.numbers((e * n, k), F32, 2, 0.1).view(e, n, k)
    dy = H.numbers((m, n), F32, 3)
    codes, scales = FB.convert_to_fp8_block(w.cuda(), is_2d_block=True)
    got = FB.fp8_block_grouped_linear(x.cuda(), codes, scales, ends.cuda())
    xl, b = x.cuda().requires_grad_(True), w.cuda().transpose(1, 2).requires_grad_(True)
    y = grouped._quantize_then_fp8_block_scaled_grouped_mm(xl, b, offs=ends.cuda())
    dx, dw = torch.autograd.grad(y, (xl, b), dy.cuda())
    at = 0
    for i, end in enumerate(ends.tolist()):
        if end > at:
            r = slice(at, end)
            xv, wv = H.quantize(x[r], "e4m3", -1)[2], H.quantize(w[i], "e4m3", None)[2]
            H.assert_within(got[r], *H.product_bound(xv, wv, F32), f"served {i}")
            H.assert_within(y[r], *H.product_bound(xv, wv, F32), f"y {i}")
            H.assert_within(dx[r], *H.product_bound(H.quantize(dy[r], "e4m3", -1)[2], wv.T, F32), f"dx {i}")
            H.assert_within(dw[i], *H.product_bound(H.quantize(x[r], "e4m3", -2)[2].T, H.quantize(dy[r], "e4m3", -2)[2].T, F32), f"dw {i}")
        at = end
    assert not bool(got[at:].any()) and not bool(y[at:].any()) and not bool(dx[at:].any())


@pytest.mark.parametrize("ends", [[300, 1047700, 1049990], [1047552, 1047552, 1047600], [1048000, 5, 2 ** 30], [0, 0, 0]], ids=str)
def test_more_rows_than_a_launch_lists(ends):
    # 4096 units of 256 rows, 1 047 552 rows here, and those behind them
    m, n, k, cut = 1_050_000, 48, 144, 500_000
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = torch.randn(m, k, device="cuda", generator=g).to(BF), torch.randn(m, n, device="cuda", generator=g).to(BF)
    w = H.numbers((3 * n, k), BF, 2, 0.1).cuda().view(3, n, k)
    codes, scales = FB.convert_to_fp8_block(w, is_2d_block=True)
    offs = torch.tensor(ends, device="cuda", dtype=torch.int32)

    def run(rows, o):
        xl = x[rows].requires_grad_(True)
        y = grouped._quantize_then_fp8_block_scaled_grouped_mm(xl, w.transpose(1, 2), offs=o)
        return FB.fp8_block_grouped_linear(x[rows], codes, scales, o), y, torch.autograd.grad(y, xl, dy[rows])[0]
    whole = run(slice(0, m), offs)
    for rows, o in ((slice(0, cut), offs.clamp(max=cut)), (slice(cut, m), in_order(offs, m).sub(cut).clamp(min=0))):
        assert all(torch.equal(a[rows], b) for a, b in zip(whole, run(rows, o)))
    at = 0
    for e, end in enumerate(in_order(offs, m).tolist()):
        rows = sorted({r for r in (at, at + 1, (at + end) // 2, 1047551, 1047552, end - 1) if at <= r < end})
        wv = H.quantize(w[e].cpu(), "e4m3", None)[2]
        for got, src, right in ((whole[0], x, wv), (whole[1], x, wv), (whole[2], dy, wv.T.contiguous())):
            H.assert_within(got[rows], *H.product_bound(H.quantize(src[rows].cpu(), "e4m3", -1)[2], right, BF))
        at = end
    assert not any(bool(t[at:].any()) for t in whole)


def test_offsets_past_thirty_two_bits():
    e, n, k = 34, 4096, 32768                                # 4.6 GB of codes
    codes = torch.empty(e, n, k, device="cuda", dtype=torch.float8_e4m3fn)
    scales = torch.empty(e, n // 128, k // 128, device="cuda")
    for i in range(e):
        w = torch.randn(n, k, device="cuda", dtype=BF, generator=torch.Generator("cuda").manual_seed(i))
        codes[i], scales[i] = FB.convert_to_fp8_block(w, is_2d_block=True)
    for counts in ([0] * 32 + [2, 3], [0] * 31 + [300, 20, 30], [0] * 33 + [400]):
        m = sum(counts)
        x = torch.randn(m, k, device="cuda", dtype=BF, generator=torch.Generator("cuda").manual_seed(99))
        got = FB.fp8_block_grouped_linear(x, codes, scales, H.runs(counts).cuda())
        at = 0
        for i, c in enumerate(counts):
            if c:
                want = FB.fp8_block_linear(x[at:at + c], codes[i], scales[i])
                size = float(want.abs().max())
                # other kernels, the same codes: sums in another order (256 blocks) and a rounding to bf16
                assert float((got[at:at + c].float() - want.float()).abs().max()) <= size * 2.0 ** -7
                at += c
    del codes, scales
    x = torch.randn(70000, 32768, device="cuda", dtype=BF)   # 2.3e9 numbers
    codes, scales = FB.convert_to_fp8_block(x)
    tail, tail_scales = FB.convert_to_fp8_block(x[-300:])
    assert torch.equal(codes[-300:].view(torch.uint8), tail.view(torch.uint8)) and torch.equal(scales[-300:], tail_scales)
    back = FB.convert_from_fp8_block(codes, scales, BF)
    assert torch.equal(back[-300:], FB.convert_from_fp8_block(tail, tail_scales, BF))
    del back
    codes, scales = FB.convert_to_fp8_block(x, axis=-2)
    tail, tail_scales = FB.convert_to_fp8_block(x[-(70000 % 128):], axis=-2)
    assert torch.equal(codes[-(70000 % 128):].contiguous().view(torch.uint8), tail.contiguous().view(torch.uint8))
    assert torch.equal(scales[-1:], tail_scales)


# ---------------------------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------------------------
def test_two_streams_at_once():
    xs = [H.numbers((m, 512), BF, m).cuda() for m in (3, 24, 500)]
    ws = [H.numbers((768, 512), BF, 7 + i, 0.1).cuda() for i in range(2)]

    def run(w):
        got = []
        for x in xs:
            c, s = FB.convert_to_fp8_block(w, is_2d_block=True)
            got.append(FB.fp8_block_linear(x, c, s))
            xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            y = FB._to_fp8_block_then_scaled_mm(xl, wl)
            got += [y.detach(), *torch.autograd.grad(y, (xl, wl), y.detach())]
        return got
    want = [run(w) for w in ws]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ws]
    for _ in range(5):
        got = []
        for s, w in zip(streams, ws):
            with torch.cuda.stream(s):
                got.append(run(w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_captured_steps_in_two_graphs_of_one_pool():
    x, w, dy = (H.numbers(s, BF, i).cuda() for i, s in enumerate(((300, 272), (144, 272), (300, 144))))
    b = H.numbers((2 * 272, 144), BF, 5).cuda().view(2, 272, 144)
    offs = torch.tensor([100, 300], device="cuda", dtype=torch.int32)
    xl, wl, bl = (t.clone().requires_grad_(True) for t in (x, w, b))

    def step():
        y = FB._to_fp8_block_then_scaled_mm(xl, wl)
        z = grouped._quantize_then_fp8_block_scaled_grouped_mm(xl, bl, offs=offs)
        c, s = FB.convert_to_fp8_block(wl, is_2d_block=True)
        few = FB.fp8_block_linear(xl.detach()[:20], c, s)
        one = FB.fp8_block_linear(xl.detach()[:1], c, s)
        return (y.detach(), z.detach(), few, one, *torch.autograd.grad((y, z), (xl, wl, bl), (dy, dy)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    # (A leaf's eager graph has to be gone: its node belongs to the stream that it was made on, and torch's engine refuses to join
    # that stream to a capture, whatever the operator.  One of other leaves may live.)
    alive = FB._to_fp8_block_then_scaled_mm(other := x.clone().requires_grad_(True), w)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g, pool=graphs[0].pool() if outs else None):
            outs.append(step())
    for seed in (11, 12):
        with torch.no_grad():
            xl.copy_(H.numbers((300, 272), BF, seed)), dy.copy_(H.numbers((300, 144), BF, seed + 5)), bl.mul_(1.25)
            offs.copy_(torch.tensor([seed, 290]))
        want = step()
        for g, out in zip(graphs, outs):
            g.replay()
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    alive.backward(dy)
    assert bool(torch.isfinite(other.grad).all())


@pytest.mark.parametrize("m", [1, 8, 9, 24, 200])
def test_weights_that_were_just_written(m):
    """What is served may have been written by the launch before: nothing is read of it too early."""
    n, k = 4096, 1024
    x = torch.randn(m, k, device="cuda", dtype=BF)
    ws = [torch.randn(n, k, device="cuda", dtype=BF) for _ in range(2)]
    pairs = [FB.convert_to_fp8_block(w, is_2d_block=True) for w in ws]
    want = [FB.fp8_block_linear(x, *p) for p in pairs]
    codes, scales = (t.clone() for t in pairs[0])
    for i in range(20):
        c, s = pairs[i % 2]
        scales.copy_(s)
        codes.copy_(c)
        a = x.mul(1.0)
        got = FB.fp8_block_linear(a, codes, scales)
        a.zero_()
        assert torch.equal(got, want[i % 2])
        codes.zero_()


@pytest.mark.parametrize("m,n,k", [(8, 4096, 1024), (300, 4096, 2048), (2000, 272, 400), (2000, 1040, 4096)])
def test_operands_that_were_just_written(m, n, k):
    """Both operands may come from the launches in front, and go right behind."""
    xs, ws = [torch.randn(m, k, device="cuda", dtype=BF) for _ in range(2)], [torch.randn(n, k, device="cuda", dtype=BF) for _ in range(2)]
    dy = torch.randn(m, n, device="cuda", dtype=BF)

    def step(x, w):
        xl, wl = x.requires_grad_(True), w.requires_grad_(True)
        y = FB._to_fp8_block_then_scaled_mm(xl, wl)
        return (y.detach(), *torch.autograd.grad(y, (xl, wl), dy))
    want = [step(x.clone(), w.clone()) for x, w in zip(xs, ws)]
    for i in range(20):
        x, w = xs[i % 2].mul(1.0), ws[i % 2].mul(1.0)
        got = step(x, w)
        with torch.no_grad():
            x.zero_(), w.zero_()
        del x, w
        assert all(torch.equal(a, b) for a, b in zip(got, want[i % 2]))


def test_copies_land_before_a_pair_that_gave_up_ends():
    """The wait behind a role that gave up, for every number of stages that the two producers can have issued (0 to 9, either up to
    four ahead); without a wait that runs out, and with the products as they were behind it."""
    from alto_b200 import _lib as L
    cases = sum(min(m, 4) + 5 for m in range(10))
    for _ in range(3):
        assert L.selftest_drain() == (0, cases)
    assert L.status_read()[0] == 0
    x, w = H.numbers((300, 528), BF, 1), H.numbers((272, 528), BF, 2, 0.1)
    exact, bound = H.product_bound(H.quantize(x, "e4m3", -1)[2], H.quantize(w, "e4m3", None)[2], BF)
    H.assert_within(FB._to_fp8_block_then_scaled_mm(x.cuda(), w.cuda()), exact, bound)


def test_results_do_not_change_from_call_to_call():
    x, w, dy = torch.randn(2000, 1040, device="cuda", dtype=BF), torch.randn(784, 1040, device="cuda", dtype=BF), torch.randn(2000, 784, device="cuda", dtype=BF)

    def step():
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = FB._to_fp8_block_then_scaled_mm(xl, wl)
        c, s = FB.convert_to_fp8_block(w, is_2d_block=True)
        return (y, *torch.autograd.grad(y, (xl, wl), dy), *(FB.fp8_block_linear(x[:m], c, s) for m in (3, 14, 31)))
    want = step()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_a_graph_that_is_used_twice_and_saved_elsewhere():
    x, w, dy = (H.numbers(s, BF, i).cuda() for i, s in enumerate(((300, 272), (144, 272), (300, 144))))
    b, offs = H.numbers((2 * 272, 144), BF, 5).cuda().view(2, 272, 144), torch.tensor([100, 290], device="cuda", dtype=torch.int32)

    def grads(twice=False, change=False):
        xl, wl, bl = (t.clone().requires_grad_(True) for t in (x, w, b))
        y = FB._to_fp8_block_then_scaled_mm(xl, wl)
        z = grouped._quantize_then_fp8_block_scaled_grouped_mm(xl, bl, offs=offs)
        if change:                       # what is kept are codes
            with torch.no_grad():
                xl.zero_(), wl.zero_(), bl.zero_()
        if twice:
            torch.autograd.grad((y, z), (xl, wl, bl), (dy, dy), retain_graph=True)
        return torch.autograd.grad((y, z), (xl, wl, bl), (dy, dy))
    want = grads()
    assert all(torch.equal(p, q) for p, q in zip(grads(twice=True), want))
    assert all(torch.equal(p, q) for p, q in zip(grads(change=True), want))
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(p, q) for p, q in zip(grads(), want))
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        grads()
    assert kept and all(t.dtype in (torch.uint8, torch.float32, torch.int32) for t in kept)


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
class GroupedExperts(nn.Module):
    def __init__(self, e, d, h):
        super().__init__()
        self.w1 = nn.Parameter(torch.randn(e, h, d) * 0.05)
        self.w2 = nn.Parameter(torch.randn(e, d, h) * 0.05)

    def forward(self, x, offs):
        h = torch._grouped_mm(x, self.w1.transpose(-2, -1), offs=offs)
        return torch._grouped_mm(torch.relu(h), self.w2.transpose(-2, -1), offs=offs)


def test_a_training_step_and_serving_of_its_weights():
    torch.manual_seed(3)
    e, d, h, rows = 4, 272, 400, 500
    model = nn.ModuleDict(dict(up=nn.Linear(d, d, bias=False), experts=GroupedExperts(e, d, h))).to("cuda", BF)
    plain = {n: p.detach().clone() for n, p in model.named_parameters()}
    LowPrecisionTrainingModifier(scheme="fp8_block_e4m3", targets=["Linear", "GroupedExperts"]).convert(model)
    offs = torch.tensor([100, 100, 349, 480], device="cuda", dtype=torch.int32)
    x, c = torch.randn(rows, d, device="cuda", dtype=BF), torch.randn(rows, d, device="cuda", dtype=BF)
    u = model.up(x)
    y = model.experts(u, offs)
    y.backward(c)
    # every layer against 64 bits, from what the layer before gave
    up = H.product_bound(H.quantize(x.cpu(), "e4m3", -1)[2], H.quantize(plain["up.weight"].cpu(), "e4m3", None)[2], BF)
    H.assert_within(u, *up, "up")
    assert not bool(y[480:].any())
    params = list(model.parameters())
    assert all(p.grad is not None and p.grad.shape == p.shape for p in params)
    grads = [p.grad.detach().clone() for p in params]
    grads = [g._data if hasattr(g, "_data") else g for g in grads]
    exact = sum(float(g.double().square().sum()) for g in grads) ** 0.5
    norm = grad_clip.clip_grad_norm_(params, exact / 3)
    # fp32 sums of 32 squares, the root and its rounding
    assert abs(float(norm) - exact) <= exact * 19 * 2.0 ** -24
    f = (exact / 3) / (exact + 1e-6)
    for p, g in zip(params, grads):
        now = p.grad._data if hasattr(p.grad, "_data") else p.grad
        # norm, factor and product in fp32, then bf16
        assert bool(((now.double() - g.double() * f).abs() <= g.double().abs() * f * (24 * 2.0 ** -24 + 2.0 ** -8) + 2.0 ** -133).all())
    before = {n: p.detach()._data.clone() for n, p in model.named_parameters()}
    torch.optim.SGD(params, lr=0.5).step()
    after = {n: p.detach()._data for n, p in model.named_parameters()}
    assert all(not torch.equal(before[n], after[n]) for n in before)
    # and served, from one token up
    with torch.no_grad():
        codes = {n: FB.convert_to_fp8_block(w, is_2d_block=True) for n, w in after.items()}
        for m in (1, 7, 30, 480):
            ends = offs.clamp(max=m)
            a = FB.fp8_block_linear(x[:m], *codes["up.weight"])
            b = torch.relu(FB.fp8_block_grouped_linear(a, *codes["experts.w1"], ends))
            got = FB.fp8_block_grouped_linear(b, *codes["experts.w2"], ends)
            at = 0
            for i, end in enumerate(ends.tolist()):
                if end > at:
                    w2 = H.quantize(after["experts.w2"][i].cpu(), "e4m3", None)[2]
                    H.assert_within(got[at:end], *H.product_bound(H.quantize(b[at:end].cpu(), "e4m3", -1)[2], w2, BF), f"expert {i} of {m}")
                at = end
            H.assert_within(a, *H.product_bound(H.quantize(x[:m].cpu(), "e4m3", -1)[2], H.quantize(after["up.weight"].cpu(), "e4m3", None)[2], BF))


def test_wrapped_weights_give_what_the_functions_give():
    x, w, dy = (H.numbers(s, BF, i).cuda() for i, s in enumerate(((60, 272), (144, 272), (60, 144))))
    p, xl, wl = wrapped(w), x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = FB._to_fp8_block_then_scaled_mm(xl, wl)
    want.backward(dy)
    for call in (lambda a: nn.functional.linear(a, p), lambda a: torch.matmul(a, p.t())):
        p.grad, a = None, x.clone().requires_grad_(True)
        y = call(a)
        y.backward(dy)
        g = p.grad._data if hasattr(p.grad, "_data") else p.grad
        assert torch.equal(y, want) and torch.equal(a.grad, xl.grad) and torch.equal(g, wl.grad)
    bias = torch.randn(144, device="cuda", dtype=BF)
    assert torch.equal(nn.functional.linear(x, p, bias), want + bias)
