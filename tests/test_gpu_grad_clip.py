"""Norm of many tensors and clipping by it, against 64 bits."""
import math

import pytest
import torch

from alto_b200 import grad_clip as GC

pytestmark = pytest.mark.gpu


def tensors(sizes, dtypes, seed=0, std=1e-2, gap=0):
    """Views of one buffer per type, one behind the other (``gap``: elements between them)."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = dtypes[i % len(dtypes)]
        out.append((torch.randn(n + gap, generator=g) * std).to(t).cuda()[gap:])
    return out


def exact_norm(ts, inf):
    if inf:
        return max([float(t.double().abs().max()) for t in ts if t.numel()] or [0.0])
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in ts))


def factor(norm, most):
    return min(1.0, most / (norm + 1e-6))


SIZES = [[1], [7, 8, 9], [0, 3, 0], [4096 * 8, 4096 * 8 + 1, 33, 65536 * 8 - 1], [1000003], list(range(1, 400)), [5] * 2500]
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("inf", [False, True])
@pytest.mark.parametrize("dtypes", [[BF], [F32], [BF, F32]], ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[-1]}")
@pytest.mark.parametrize("gap", [0, 1])
def test_norm_and_clipping(sizes, dtypes, inf, gap):
    ts = tensors(sizes, dtypes, len(sizes), gap=gap)
    before = [t.clone() for t in ts]
    kind = math.inf if inf else 2.0
    exact = exact_norm(ts, inf)
    # the root and its rounding to fp32: 2^-24 each; fp32 sums of at most 32 squares, 33 roundings of 2^-24 of the square, half of it
    # in the root
    near = exact * (33 / 2 + 2) * 2.0 ** -24
    assert abs(float(GC.grad_norm(ts, kind)) - exact) <= near
    most = exact * 0.37
    into = [torch.full_like(t, 7.0) for t in ts]
    norm = GC.clip_grads(ts, most, kind, out=into)
    assert norm.dtype == F32 and norm.dim() == 0 and abs(float(norm) - exact) <= near
    f = factor(exact, most)
    for t, b, o in zip(ts, before, into):
        assert torch.equal(t, b)                    # only out is written
        want = b.double() * f
        # norm, factor and product rounded to fp32 steps, then to the type
        bound = want.abs() * ((33 / 2 + 6) * 2.0 ** -24 + (2.0 ** -8 if t.dtype == BF else 2.0 ** -24)) + 2.0 ** -133
        assert bool(((o.double() - want).abs() <= bound).all())
    again = GC.clip_grads(ts, most, kind)           # in place: the same bits
    assert torch.equal(again, norm) and all(torch.equal(t, o) for t, o in zip(ts, into))
    held = [t.clone() for t in ts]
    GC.clip_grads(ts, exact * 4, kind)              # nothing to clip
    assert all(torch.equal(t, b) for t, b in zip(ts, held))
    copied = [torch.full_like(t, 7.0) for t in ts]
    GC.clip_grads(ts, exact * 4, kind, out=copied)
    assert all(torch.equal(t, b) for t, b in zip(copied, held))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("std", [1e30, 1e-30, 1e-38, 0.0])
def test_far_from_one(std, dtype):
    ts = [t.to(dtype) for t in tensors([70001, 13], [F32], 3, std)]
    exact = exact_norm(ts, False)
    got = float(GC.grad_norm(ts))
    assert abs(got - exact) <= exact * (33 / 2 + 2) * 2.0 ** -24
    mixed = tensors([5000], [F32], 4, 1e-3) + ts
    exact = exact_norm(mixed, False)
    assert abs(float(GC.grad_norm(mixed)) - exact) <= exact * (33 / 2 + 2) * 2.0 ** -24


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("where", [0, 3, 50000, 70000])
def test_not_finite(where, kind, bad):
    for dtype in (BF, F32):
        ts = tensors([11, 70001], [dtype])
        ts[1][where] = bad
        norm = float(GC.grad_norm(ts, kind))
        assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
        before = [t.clone() for t in ts]
        with pytest.raises(RuntimeError, match="non-finite"):
            GC.clip_grads(ts, 1.0, kind, error_if_nonfinite=True)
        assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(ts, before))
        GC.clip_grads(ts, 1.0, kind)
        want = torch.nn.utils.clip_grads_with_norm_
        ps = [torch.nn.Parameter(b.clone()) for b in before]
        for p, b in zip(ps, before):
            p.grad = b.clone()
        want(ps, 1.0, torch.tensor(norm, device="cuda"))
        assert all(torch.equal(a.isnan(), p.grad.isnan()) and torch.equal(a.nan_to_num(5.0), p.grad.nan_to_num(5.0)) for a, p in zip(ts, ps))


def test_parameters_and_layouts():
    g = torch.Generator().manual_seed(1)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g).cuda()) for s in ((64, 48), (5,), (7, 9, 11), (3, 1))]
    grads = [torch.randn(48, 64, generator=g).cuda().t(), torch.randn(10, generator=g).cuda()[::2], torch.randn(7, 9, 22, generator=g).cuda()[..., ::2],
             None]
    for p, q in zip(ps, grads):
        p.grad = q
    before = [q.clone() for q in grads[:3]]
    exact = exact_norm(before, False)
    norm = GC.clip_grad_norm_(ps, 0.5)
    assert abs(float(norm) - exact) <= exact * 19 * 2.0 ** -24
    f = factor(exact, 0.5)
    for p, b in zip(ps, before):
        assert bool(((p.grad.double() - b.double() * f).abs() <= b.double().abs() * f * 25 * 2.0 ** -24).all())
    assert float(GC.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3).cuda())], 1.0)) == 0.0
    p = torch.nn.Parameter(torch.zeros(4).cuda())
    p.grad = torch.full((4,), 3.0, device="cuda")
    assert float(GC.clip_grad_norm_(p, 3.0)) == 6.0
    assert bool(((p.grad - 1.5).abs() < 1e-5).all())
    out = [torch.zeros(48, 64).cuda().t(), torch.zeros(64, 48).cuda()]      # other strides than the gradients'
    src = [grads[0], grads[0]]
    GC.clip_grads(src, 1e9, out=out)
    assert torch.equal(out[0], src[0]) and torch.equal(out[1], src[0])


def test_captured_and_replayed():
    ts = tensors([70001, 5, 3000], [BF, F32])
    into = [torch.empty_like(t) for t in ts]
    GC.clip_grads(ts, 1.0, out=into)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = GC.clip_grads(ts, 0.1, out=into)
    for k in range(3):
        for t in ts:
            t.mul_(1.5)
        graph.replay()
        want = [torch.empty_like(t) for t in ts]
        n = GC.clip_grads(ts, 0.1, out=want)
        assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(into, want))


def test_a_tensor_that_is_listed_twice_and_versions():
    t, u = tensors([70001, 5], [F32])
    before = t.clone()
    for bad, out in (([t, u, t], None), ([t, t.view(-1)], None), ([t, t], [u.new_empty(70001)] * 2)):
        with pytest.raises(ValueError, match="twice"):
            GC.clip_grads(bad, 1e-3, out=out)
    assert torch.equal(t, before)
    empty = t[:0]
    GC.clip_grads([empty, empty, u], 1e-3)
    # a graph that holds what is written says so
    leaf = torch.randn(100, device="cuda").requires_grad_(True)
    g = torch.randn(100, device="cuda")
    y = leaf * g
    GC.clip_grads([g], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        GC.clip_grads([torch.randn(100, device="cuda")], 1e-3)


def test_gradients_that_others_are_scaled_into():
    flat = torch.randn(64, device="cuda")
    a, b, c, d = (flat[16 * i:16 * i + 16] for i in range(4))
    before = flat.clone()
    for grads, out in (([a, b], [b, a]), ([a, b], [c, a]), ([a, b, c], [d, b, a]), ([a, b.view(4, 4).t()], [c, a.view(4, 4).t()])):
        with pytest.raises(ValueError, match="in its own place"):
            GC.clip_grads(grads, 1e-3, out=out)
    assert torch.equal(flat, before)
    norm = GC.clip_grads([a, b, c], 1e-3, out=[a, d, c])          # in its own place, or into another
    f = factor(float(norm), 1e-3)
    assert torch.equal(b, before[16:32])
    for got, src in ((a, before[:16]), (d, before[16:32]), (c, before[32:48])):
        assert bool(((got.double() - src.double() * f).abs() <= src.double().abs() * f * 25 * 2.0 ** -24).all())


def test_tensors_that_overlap_themselves():
    t, one = torch.randn(16, device="cuda"), torch.randn(4, 1, device="cuda")
    before, version = t.clone(), t._version
    spread = one.expand(4, 5)
    for grads, out in (([t, spread], None), ([t, one.repeat(1, 5)], [torch.empty_like(t), spread])):
        with pytest.raises(RuntimeError, match="single memory location"):
            GC.clip_grads(grads, 1e-3, out=out)
        assert torch.equal(t, before) and t._version == version          # nothing was scaled before
    into = [torch.empty_like(t), torch.empty(4, 5, device="cuda")]
    norm = GC.clip_grads([t, spread], 1e-3, out=into)
    assert abs(float(norm) - exact_norm([t, spread], False)) <= 1e-5
    assert torch.equal(into[1], into[1][:, :1].expand(4, 5))


def test_refusals():
    t = torch.ones(8, device="cuda")
    for bad, kind in (([t.half()], TypeError), ([t, t.cpu()], RuntimeError), ([t.to_sparse()], ValueError), ([t.long()], TypeError), ([t, None], TypeError)):
        with pytest.raises(kind):
            GC.grad_norm(bad)
        with pytest.raises(kind):
            GC.clip_grads(bad, 1.0)
    for out in ([], [t, t], [t[:4]], [t.bfloat16()], [t.view(2, 4)]):
        with pytest.raises(ValueError):
            GC.clip_grads([t], 1.0, out=out)
    assert bool((t == 1).all())


@pytest.mark.parametrize("most", [0.0, 1e-30, math.inf])
def test_extreme_limits(most):
    ts = tensors([1000, 33], [BF, F32])
    before = [t.clone() for t in ts]
    norm = GC.clip_grads(ts, most)
    if most == math.inf:
        assert all(torch.equal(a, b) for a, b in zip(ts, before))
    else:
        f = most / (float(norm) + 1e-6)
        assert all(bool(((a.double() - b.double() * f).abs() <= b.double().abs() * f * 2.0 ** -7 + 2.0 ** -133).all()) for a, b in zip(ts, before))


def test_on_another_stream_and_two_at_once():
    lists = [tensors([70001, 5, 300000], [BF, F32], seed=i) for i in range(2)]
    want = [[t.clone() for t in l] for l in lists]
    norms = [GC.clip_grads(l, 0.1) for l in want]
    streams = [torch.cuda.Stream() for _ in lists]
    torch.cuda.synchronize()
    got = []
    for s, l in zip(streams, lists):
        with torch.cuda.stream(s):
            got.append(GC.clip_grads(l, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, norms))
    assert all(torch.equal(a, b) for l, w in zip(lists, want) for a, b in zip(l, w))


def test_sharded_tensors_of_a_mesh_of_one():
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Replicate, Shard
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cuda", (1,))
        ts = tensors([70001, 5, 300000, 0], [BF, F32])
        want = [t.clone() for t in ts]
        norm = GC.clip_grads(want, 0.1)
        sharded = [DTensor.from_local(t.clone(), mesh, [Shard(0) if i % 2 else Replicate()]) for i, t in enumerate(ts)]
        into = [torch.zeros_like(t) for t in sharded]
        for out in (into, None):
            got = GC.clip_grads(sharded, 0.1, out=out)
            assert type(got) is torch.Tensor and abs(float(got) - float(norm)) <= 4e-7 * float(norm)
            # (sums of types that are apart have another order: a factor that is off by steps of fp32)
            assert all(torch.allclose(a.to_local().double(), b.double(), rtol=2.0 ** -7 if b.dtype == BF else 1e-6, atol=0)
                       for a, b in zip(out or sharded, want))
        mixed = [ts[0].clone(), DTensor.from_local(ts[1].clone(), mesh, [Shard(0)])]
        assert abs(float(GC.grad_norm(mixed, math.inf)) - exact_norm(ts[:2], True)) == 0.0
        with pytest.raises(TypeError):
            GC.clip_grads([DTensor.from_local(torch.ones(3, device="cuda").half(), mesh, [Shard(0)])], 1.0)
    finally:
        dist.destroy_process_group()


def test_nothing_in_the_list_and_long_tensors():
    empty = [torch.empty(0, device="cuda"), torch.empty(0, 5, device="cuda", dtype=BF)]
    assert float(GC.grad_norm(empty)) == 0.0 and float(GC.clip_grads(empty, 1.0)) == 0.0 and float(GC.clip_grads(empty, 1.0, math.inf)) == 0.0
    t = torch.zeros(2 ** 31 + 70001, device="cuda", dtype=BF)
    u = torch.zeros(2 ** 31 + 9, device="cuda", dtype=BF)[1:]          # off 16 bytes
    t[5], t[-3], u[2 ** 31], u[7] = 1.0, 2.0, 2.0, 4.0
    assert float(GC.grad_norm([t, u])) == 5.0 and float(GC.grad_norm([t, u], math.inf)) == 4.0
    assert float(GC.clip_grads([t, u], 2.5)) == 5.0
    half = 2.5 / (5.0 + 1e-6)
    for got, want in ((t[5], 1.0), (t[-3], 2.0), (u[2 ** 31], 2.0), (u[7], 4.0)):
        assert abs(float(got) - want * half) <= want * half * (2.0 ** -8 + 2.0 ** -23)
    assert int(torch.count_nonzero(t)) == 2 and int(torch.count_nonzero(u)) == 2
