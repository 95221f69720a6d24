"""Norms and clipping of sharded gradients, as gloo ranks: what is summed over which ranks.  The kernels' part is restated on the
CPU; it takes plain tensors alone, as they do."""
import math
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch.distributed.device_mesh import init_device_mesh
from torch.distributed.tensor import DTensor, Partial, Replicate, Shard, distribute_tensor

from alto_b200 import _lib as L
from alto_b200 import grad_clip as GC


class Host:
    """``_autograd.so``'s two functions in elementary operations."""

    @staticmethod
    def _plain(ts):
        return len(ts) > 0 and all(type(t) in (torch.Tensor, torch.nn.Parameter) for t in ts)

    def grad_norm(self, ts, inf):
        if not self._plain(ts):
            return None
        with torch.no_grad():
            flat = torch.cat([t.double().flatten() for t in ts])
            total = (flat.abs().amax() if flat.numel() else flat.sum()) if inf else flat.square().sum()
        return total, (total if inf else total.sqrt()).float()

    def clip_grads(self, grads, outs, most, inf, total):
        if not self._plain(grads) or (outs and (not self._plain(outs) or any(o.shape != g.shape for o, g in zip(outs, grads)))):
            return None
        total = self.grad_norm(grads, inf)[0] if total is None else total
        norm = total if inf else total.sqrt()
        f = (most / (norm + 1e-6)).clamp_max(1.0).float()
        with torch.no_grad():
            for g, o in zip(grads, outs or grads):
                o.copy_(g * f)
        return norm.float()


def over_ranks(fn, world):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_rank, args=(fn, world, port), nprocs=world, join=True)


def _rank(rank, fn, world, port):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.set_num_threads(1)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    L._autograd_module = Host()
    try:
        fn(rank)
    finally:
        dist.destroy_process_group()


def numbers(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def exact(ts, inf):
    return max(float(t.abs().max()) for t in ts) if inf else math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def check(tensors, full, group=None):
    """Norm, clipping into others and in place, of tensors that stand for ``full`` on every rank."""
    for inf in (False, True):
        kind, want = (math.inf if inf else 2.0), exact(full, inf)
        assert abs(float(GC.grad_norm(tensors, kind, group=group)) - want) <= 1e-6 * want
        f = min(1.0, 0.25 * want / (want + 1e-6))
        whole = lambda ts: [t.full_tensor() if isinstance(t, DTensor) else t for t in ts]      # noqa: E731
        before, out = whole(tensors), [torch.zeros_like(t) for t in tensors]
        norm = GC.clip_grads(tensors, 0.25 * want, kind, out=out, group=group)
        assert type(norm) is torch.Tensor and norm.dtype == torch.float32 and abs(float(norm) - want) <= 1e-6 * want
        assert all(torch.equal(a, b) for a, b in zip(whole(tensors), before))
        assert all(torch.allclose(a, b * f, rtol=1e-6, atol=0) for a, b in zip(whole(out), full))
        params = [torch.nn.Parameter(torch.zeros_like(t)) for t in tensors]
        for p, t in zip(params, tensors):
            p.grad = t.clone()
        versions = [p.grad._version for p in params]
        norm = GC.clip_grad_norm_(params, 0.25 * want, kind, group=group, error_if_nonfinite=True)
        assert abs(float(norm) - want) <= 1e-6 * want
        got = [p.grad for p in params]
        assert all(torch.allclose(a, b * f, rtol=1e-6, atol=0) for a, b in zip(whole(got), full))
        assert all(t._version > v for t, v in zip(got, versions))


def _one_dimension(rank):
    mesh, world = init_device_mesh("cpu", (2,)), dist.group.WORLD
    full = [numbers(5, 4, seed=1), numbers(1, 3, seed=2), numbers(6, 8, seed=3), numbers(7, seed=4)]
    even, short, cols = (distribute_tensor(t, mesh, [Shard(d)]) for t, d in zip(full, (0, 0, 1)))      # (of the second, rank 1 has nothing)
    copies = distribute_tensor(full[3], mesh, [Replicate()])
    check([even, short, cols], full[:3])
    check([even], full[:1])
    check([copies], full[3:])                         # once, not once a rank
    check([copies, even, cols, short], [full[3], full[0], full[2], full[1]])
    check([full[3].clone(), even], [full[3], full[0]])
    check([even, short, cols], full[:3], world)       # over the mesh's own ranks, said by the caller
    both = [full[3][rank * 4:rank * 4 + 4], even]     # parts of everything
    assert abs(float(GC.grad_norm(both, group=world)) - exact([full[3], full[0]], False)) <= 1e-5
    # a NaN in one part is everyone's
    bad = DTensor.from_local(torch.full((2, 2), float("nan") if rank else 1.0), mesh, [Shard(0)])
    for kind in (2.0, math.inf):
        assert math.isnan(float(GC.grad_norm([copies, bad], kind)))
        with pytest.raises(RuntimeError, match="non-finite"):
            GC.clip_grads([copies, bad], 1.0, kind, error_if_nonfinite=True)
    partial = DTensor.from_local(torch.ones(2), mesh, [Partial()])
    for call in (lambda: GC.grad_norm([copies], group=world), lambda: GC.clip_grads([even, copies], 1.0, group=world),
                 lambda: GC.grad_norm([even, partial]), lambda: GC.clip_grads([partial], 1.0), lambda: GC.clip_grads([partial], 1.0, group=world),
                 lambda: GC.clip_grads([even], 1.0, out=[torch.zeros_like(even.to_local())]),
                 lambda: GC.clip_grads([copies], 1.0, out=[DTensor.from_local(torch.zeros(7), mesh, [Shard(0)])])):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(even.full_tensor(), full[0]) and torch.equal(copies.full_tensor(), full[3])


def _a_rank_without_tensors(rank):
    world = dist.group.WORLD
    for empty in (0, 1):
        for inf in (False, True):
            kind = math.inf if inf else 2.0
            for value in (numbers(9, seed=1), torch.zeros(4), torch.empty(0), torch.tensor([1.0, math.nan]), torch.tensor([math.inf])):
                ts = [] if rank == empty else [value.clone()]
                want = exact([value], inf) if value.numel() and not value.isnan().any() else math.nan if value.numel() else 0.0
                same = lambda got: got.dtype == torch.float32 and got.dim() == 0 and (          # noqa: E731
                    float(got) == pytest.approx(want, rel=1e-6, nan_ok=True))
                assert same(GC.grad_norm(ts, kind, group=world))
                assert same(GC.clip_grads(ts, 0.5, kind, out=[t.clone() for t in ts], group=world))
                if not math.isfinite(want):
                    with pytest.raises(RuntimeError, match="non-finite"):
                        GC.clip_grads(ts, 0.5, kind, group=world, error_if_nonfinite=True)
                assert same(GC.clip_grads(ts, 0.5, kind, group=world))          # in place
        used = torch.nn.Parameter(torch.zeros(9))
        if rank != empty:
            used.grad = numbers(9, seed=2)
        want = exact([numbers(9, seed=2)], False)
        assert abs(float(GC.clip_grad_norm_([used], 0.5, group=world)) - want) <= 1e-6 * want
        assert (used.grad is None) == (rank == empty)
    for call in (lambda: GC.grad_norm([], group=world), lambda: GC.clip_grads([], 1.0, group=world), lambda: GC.clip_grads([], 1.0, out=[], group=world)):
        with pytest.raises(ValueError, match="on one of them at least"):
            call()
    with pytest.raises(ValueError):          # (before anything is waited for)
        GC.clip_grads([], 1.0, out=[torch.zeros(3)], group=world)


def _two_dimensions(rank):
    mesh = init_device_mesh("cpu", (2, 2), mesh_dim_names=("replicas", "parts"))
    full = [numbers(5, 4, seed=1), numbers(6, 7, seed=2), numbers(3, seed=3), numbers(8, 2, seed=4)]
    hybrid = distribute_tensor(full[0], mesh, [Replicate(), Shard(0)])
    every = distribute_tensor(full[1], mesh, [Shard(0), Shard(1)])
    first = distribute_tensor(full[2], mesh, [Shard(0), Replicate()])
    inner = distribute_tensor(full[3], mesh["parts"], [Shard(0)])            # a mesh of its own, over the same ranks
    check([hybrid, every, first, inner], full)
    check([hybrid, inner], [full[0], full[3]], mesh.get_group("parts"))
    for bad in (every, first):
        with pytest.raises(ValueError, match="parts lie on"):
            GC.grad_norm([bad], group=mesh.get_group("parts"))
    check([every], full[1:2], dist.group.WORLD)
    with pytest.raises(ValueError, match="parts lie on"):
        GC.clip_grads([hybrid], 1.0, group=dist.group.WORLD)


def _sharded_model(rank):
    """Gradients as fully_shard leaves them, over two dimensions with tensor parallelism (a shard of a shard)."""
    from torch.distributed.fsdp import fully_shard
    from torch.distributed.tensor.parallel import ColwiseParallel, parallelize_module
    mesh = init_device_mesh("cpu", (2, 2), mesh_dim_names=("data", "model"))
    torch.manual_seed(5)
    plain = torch.nn.Sequential(torch.nn.Linear(6, 8), torch.nn.Linear(8, 4))
    model = torch.nn.Sequential(torch.nn.Linear(6, 8), torch.nn.Linear(8, 4))
    model.load_state_dict(plain.state_dict())
    parallelize_module(model[0], mesh["model"], ColwiseParallel(output_layouts=Replicate()))
    fully_shard(model, mesh=mesh["data"])
    x = numbers(3, 6, seed=6)
    plain(x).square().sum().backward()
    model(x).square().sum().backward()
    want = float(torch.nn.utils.get_total_norm([p.grad for p in plain.parameters()]))
    norm = GC.clip_grad_norm_(model.parameters(), 0.5 * want)
    assert abs(float(norm) - want) <= 1e-5 * want
    assert any(not p.is_shard() and not p.is_replicate() for q in model.parameters() for p in q.grad.placements)
    for p, q in zip(plain.parameters(), model.parameters()):
        assert torch.allclose(q.grad.full_tensor(), p.grad * 0.5, rtol=1e-4, atol=1e-7)


@pytest.mark.parametrize("fn,world", [(_one_dimension, 2), (_a_rank_without_tensors, 2), (_two_dimensions, 4), (_sharded_model, 4)], ids=lambda v: getattr(v, "__name__", str(v)))
def test_sharded_gradients(fn, world):
    over_ranks(fn, world)
