"""Root-mean-square norm against its definition in 64 bits.

Tolerances: a result of type T is off by half a step (2^-8 of itself in bf16, 2^-24 in fp32) plus what fp32 sums leave.  A sum over
`cols` runs over at most cols / 256 + 8 terms in sequence (element-wise kernels) or 32 (vector kernels) and ten levels of
a tree; its relative error, halved by the square root, the reciprocal root's two steps and two products stay below
S = (cols / 256 + 64) 2^-24."""
import pytest
import torch

from alto_b200 import mxfp8, norm

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
EPS = 1e-5


def _inputs(rows, cols, dtype, wdtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape, std=1.0, mean=0.0, dt=dtype):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)
    return t(rows, cols, std=scale), t(rows, cols, std=2 * scale), t(cols, std=0.2, mean=1.0, dt=wdtype), t(rows, cols), t(rows, cols)


def _forward64(r, w, eps=EPS):
    d = r.double()
    root = torch.sqrt(d.pow(2).mean(-1, keepdim=True) + eps)
    return d / root, root, d / root * w.double()


def _backward64(r, w, dy, ds, eps=EPS):
    xhat, root, _ = _forward64(r, w, eps)
    gw = dy.double() * w.double()
    mean = (gw * xhat).mean(-1, keepdim=True)
    dr = (gw - xhat * mean) / root
    size = (gw.abs() + xhat.abs() * (gw * xhat).abs().mean(-1, keepdim=True)) / root
    if ds is not None:
        dr = dr + ds.double()
    return dr, size, (dy.double() * xhat).sum(0), (dy.double() * xhat).abs().sum(0)


def _sums(cols):
    return (cols / 256 + 64) * 2.0 ** -24


def _check_forward(y, r, w, eps=EPS):
    want = _forward64(r, w, eps)[2]
    assert ((y.double() - want).abs() <= want.abs() * (HALF[y.dtype] + _sums(r.shape[-1])) + 1e-37).all()


def _check_backward(dx, dw, r, w, dy, ds, eps=EPS):
    rows, cols = r.shape
    dr, size, sw, sw_size = _backward64(r, w, dy, ds, eps)
    assert ((dx.double() - dr).abs() <= dr.abs() * HALF[dx.dtype] + size * 4 * _sums(cols) + 1e-37).all()
    if dw is not None:
        assert ((dw.double() - sw).abs() <= sw.abs() * HALF[dw.dtype] + sw_size * (_sums(cols) + (rows + 32) * 2.0 ** -24)).all()


SIZES = [(1, 1), (3, 7), (5, 32), (1, 64), (130, 96), (7, 264), (33, 1000), (64, 1024), (9, 1032), (65, 2880), (31, 4096), (3, 8200),
         (2, 16384), (2, 32768), (2, 40000), (700, 512), (0, 64), (1001, 128), (77, 56), (13, 200), (1300, 255), (21, 3001),
         (6, 8191), (3, 9001), (1001, 264), (603, 4096)]


@pytest.mark.parametrize("dtype, wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                           (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("rows, cols", SIZES)
def test_norm_and_gradient(rows, cols, dtype, wdtype):
    x, res, w, dy, ds = _inputs(rows, cols, dtype, wdtype)
    x.requires_grad_(True), w.requires_grad_(True), res.requires_grad_(True)
    y = norm.rms_norm(x, w, EPS)
    assert y.dtype == dtype and y.shape == x.shape
    _check_forward(y.detach(), x.detach(), w.detach())
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dw.dtype == wdtype
    _check_backward(dx, dw, x.detach(), w.detach(), dy, None)
    y, r = norm.rms_norm(x, w, EPS, residual=res)
    assert torch.equal(r.detach(), (x.detach().float() + res.detach().float()).to(dtype))
    _check_forward(y.detach(), r.detach(), w.detach())
    dx, dres, dw = torch.autograd.grad((y, r), (x, res, w), (dy, ds))
    assert torch.equal(dx, dres)
    _check_backward(dx, dw, r.detach(), w.detach(), dy, ds)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [64, 1056, 8192, 12320])
@pytest.mark.parametrize("pitch, first", [(8, 0), (5, 0), (64, 8), (64, 3)])
def test_rows_of_a_wider_buffer(dtype, pitch, first, cols):
    rows = 37
    x, res, w, dy, ds = _inputs(rows, cols + pitch + first, dtype, dtype)
    x, res, dy, ds, w = (t[..., first:first + cols] for t in (x, res, dy, ds, w))
    x, res = x.requires_grad_(True), res.requires_grad_(True)
    y, r = norm.rms_norm(x, w, EPS, residual=res)
    _check_forward(y.detach(), r.detach(), w)
    dx, dres = torch.autograd.grad((y, r), (x, res), (dy, ds))
    _check_backward(dx, None, r.detach(), w, dy, ds)
    codes, scales, r2 = norm.rms_norm_mxfp8(x.detach(), w, EPS, residual=res.detach())
    want = mxfp8.convert_to_mxfp8(y.detach())
    assert torch.equal(r2, r) and torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])


def test_leading_dimensions_transposed_and_broadcast_rows():
    x, _, w, dy, _ = _inputs(24, 512, torch.bfloat16, torch.bfloat16)
    for view in (x.view(2, 3, 4, 512), x.view(4, 6, 512).transpose(0, 1), x.t().contiguous().t(), x[:1].expand(24, 512), x[0]):
        y = norm.rms_norm(view, w)
        assert y.shape == view.shape and torch.equal(y, norm.rms_norm(view.contiguous(), w))
    leaf = x.clone().requires_grad_(True)
    norm.rms_norm(leaf.view(4, 6, 512).transpose(0, 1), w).sum().backward()      # an upstream gradient without strides
    again = x.clone().requires_grad_(True)
    norm.rms_norm(again, w).backward(torch.ones_like(dy))
    assert torch.equal(leaf.grad, again.grad)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows, cols", [(1, 32), (3, 64), (130, 96), (17, 1024), (33, 2880), (8, 4096), (2, 16384), (2, 33024), (0, 64), (301, 128),
                                        (4, 8192), (1001, 288), (603, 2880)])
def test_mxfp8_result_is_the_quantised_norm(rows, cols, dtype, fmt):
    x, res, w, _, _ = _inputs(rows, cols, dtype, dtype)
    if rows > 1:      # rows of zeros, of infinities and NaN, of magnitudes at both ends
        x[0], res[0] = 0, 0
        x[1, 0] = float("inf")
    if rows > 2:
        x[2, cols // 2] = float("nan")
    if rows > 16:
        x[3] *= 1e-30
        x[4] *= 1e15
        w[:32] *= 1e-38
        w[32:64] *= 1e30
    for residual in (None, res):
        if rows == 0:
            got = norm.rms_norm_mxfp8(x, w, EPS, residual=residual, mxfp_format=fmt)
            assert got[0].shape == x.shape and got[1].shape == (0, cols // 32)
            continue
        y = norm.rms_norm(x, w, EPS, residual=residual)
        got = norm.rms_norm_mxfp8(x, w, EPS, residual=residual, mxfp_format=fmt)
        if residual is not None:
            assert torch.equal(got[2].view(torch.uint8), y[1].view(torch.uint8))
            y = y[0]
        codes, scales = mxfp8.convert_to_mxfp8(y, mxfp_format=fmt)
        assert got[0].dtype == codes.dtype and torch.equal(got[1], scales)
        assert torch.equal(got[0].view(torch.uint8), codes.view(torch.uint8))


def test_rows_of_zeros_infinities_and_nan_stay_by_themselves():
    x, _, w, dy, _ = _inputs(6, 2048, torch.bfloat16, torch.bfloat16)
    clean = norm.rms_norm(x, w)
    bad = x.clone()
    bad[1], bad[2, 5], bad[3, 7] = 0, float("nan"), float("inf")
    y = norm.rms_norm(bad, w)
    assert (y[1] == 0).all() and torch.isnan(y[2]).all() and torch.isnan(y[3, 7]) and (y[3, :7] == 0).all()
    assert torch.equal(y[[0, 4, 5]], clean[[0, 4, 5]])
    leaf = bad.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(norm.rms_norm(leaf, w), leaf, dy)
    _check_backward(dx[[0, 1, 4, 5]], None, bad[[0, 1, 4, 5]], w, dy[[0, 1, 4, 5]], None)


def test_gradients_that_are_not_asked_for_and_streams_alone():
    x, res, w, dy, ds = _inputs(40, 768, torch.bfloat16, torch.float32)
    w.requires_grad_(True)
    y, r = norm.rms_norm(x, w, EPS, residual=res)
    (dw,) = torch.autograd.grad(y, w, dy)
    _check_backward(torch.zeros(0, 768, device="cuda"), None, r[:0], w, dy[:0], None)
    x.requires_grad_(True)
    y, r = norm.rms_norm(x, w, EPS, residual=res)
    dx, dw2 = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(dw, dw2)
    _check_backward(dx, dw, r.detach(), w.detach(), dy, None)
    y, r = norm.rms_norm(x, w, EPS, residual=res)
    dx, dw0 = torch.autograd.grad(r, (x, w), ds)
    assert torch.equal(dx, ds) and (dw0 == 0).all()


def test_gradient_against_differences():
    x, res, w, dy, ds = _inputs(9, 160, torch.float32, torch.float32)
    x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(norm.rms_norm(x, w, EPS, residual=res), (x, w), (dy, ds))
    r, step = (x + res).detach().double(), 1e-4

    def value(a, b):
        return (_forward64(a, b)[2] * dy.double()).sum() + (a * ds.double()).sum()
    g = torch.Generator(device="cuda").manual_seed(5)
    for _ in range(4):
        v, u = torch.randn(9, 160, generator=g, device="cuda").double(), torch.randn(160, generator=g, device="cuda").double()
        along = (value(r + step * v, w.detach().double() + step * u) - value(r - step * v, w.detach().double() - step * u)) / (2 * step)
        got = (dx.double() * v).sum() + (dw.double() * u).sum()
        # r itself is rounded to fp32 (2^-24 of |r|, to first order in the slope), the difference is off by step^2
        assert abs(got - along) <= 1e-5 * (dx.double().norm() * v.norm() + dw.double().norm() * u.norm())


def test_a_second_derivative_is_refused():
    x, _, w, dy, _ = _inputs(8, 64, torch.float32, torch.float32)
    x.requires_grad_(True)
    dy.requires_grad_(True)
    (dx,) = torch.autograd.grad(norm.rms_norm(x, w), x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_captured_calls_replay_on_new_contents_and_sums_keep_their_order():
    x, res, w, dy, ds = _inputs(300, 1536, torch.bfloat16, torch.float32)
    leaf = x.clone().requires_grad_(True)
    wl = w.clone().requires_grad_(True)

    def step():
        y, r = norm.rms_norm(leaf, wl, EPS, residual=res)
        return (y.detach(), r.detach(), *torch.autograd.grad((y, r), (leaf, wl), (dy, ds)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        x2, res2, _, dy2, ds2 = _inputs(300, 1536, torch.bfloat16, torch.float32, seed)
        with torch.no_grad():
            leaf.copy_(x2), res.copy_(res2), dy.copy_(dy2), ds.copy_(ds2)
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        assert not torch.equal(got[0], first[0])


def test_refusals():
    x, res, w, _, _ = _inputs(4, 64, torch.bfloat16, torch.bfloat16)
    for bad in (dict(residual=res[:3]), dict(residual=res.float()), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            norm.rms_norm(x, w, **bad)
    with pytest.raises(ValueError):
        norm.rms_norm(x, w[:63])
    with pytest.raises(TypeError):
        norm.rms_norm(x.half(), w)
    with pytest.raises(TypeError):
        norm.rms_norm(x, w.half())
    with pytest.raises(ValueError):
        norm.rms_norm_mxfp8(x[:, :48], w[:48])
    with pytest.raises(ValueError):
        norm.rms_norm_mxfp8(x, w, mxfp_format="e3m4")
