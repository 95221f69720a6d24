"""Norm of all gradients together, and clipping by it: the step between the backward pass (or
``distributed.allreduce_gradients``) and the optimizer.

    grad_norm(tensors, norm_type)                             norm of the tensors as one vector
    clip_grad_norm_(parameters, max_norm, ...)                torch.nn.utils' function of the same name, gradients in place
    clip_grads(grads, max_norm, ..., out=...)                 the same for a list of tensors, in place or into others

    norm = sqrt(sum g^2), or max |g|          g <- g * min(1, max_norm / (norm + 1e-6))

Two launches for a thousand tensors, whatever their types (bf16, fp32), sizes and alignments; the host is not waited for.
Squares are summed in fp32 over 32 numbers and in fp64 beyond, in an order that does not change from call to call.

The reference's trainer clips with torch's function between its optimizer hooks (alto/components/optimizer.py)."""
from __future__ import annotations

import math
from typing import Iterable, Optional, Sequence, Union

import torch

from . import _lib as L
from .nvfp4 import unwrap_weight_wrapper

__all__ = ["grad_norm", "clip_grad_norm_", "clip_grads"]

_TYPES = (torch.bfloat16, torch.float32)


def _kind(norm_type) -> bool:
    """Whether the norm is the largest magnitude."""
    p = float(norm_type)
    if p == 2.0:
        return False
    if p == math.inf:
        return True
    raise ValueError(f"the norms are 2 and inf, got {norm_type}")


def _list(tensors) -> list:
    return tensors if type(tensors) is list else list(tensors)


def _refuse(name: str, tensors: Sequence[torch.Tensor], out: Sequence[torch.Tensor] = ()) -> None:
    """Says what is wrong with a list that the kernels do not take."""
    for t in (*tensors, *out):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} expects tensors, got {type(t).__name__}")
        if t.layout is not torch.strided:
            raise ValueError(f"{name} expects dense tensors, got {t.layout}")
        if not t.is_cuda:
            raise RuntimeError(f"{name} runs on CUDA tensors only (no CPU fallback)")
        if t.dtype not in _TYPES:
            raise TypeError(f"{name} expects bfloat16 or float32, got {t.dtype}")
        if t.device != tensors[0].device:
            raise ValueError(f"{name} expects all tensors on one device")
    raise ValueError(f"{name} expects out like grads: as many tensors, of their shapes and types")


def _local(t: torch.Tensor) -> torch.Tensor:
    """The local part of a sharded tensor, a wrapper's data."""
    t = t.to_local() if hasattr(t, "to_local") else t
    return unwrap_weight_wrapper(t) if hasattr(t, "_data") else t


def _sharded(t) -> bool:
    return hasattr(t, "placements") and hasattr(t, "device_mesh")


def _holders(name: str, t: torch.Tensor, group) -> tuple:
    """The process groups over whose ranks a tensor's parts lie, one behind the other: of a sharded tensor the mesh says them, and
    ``group`` has to be of the same ranks; any other tensor is a part of ``group``'s, or whole where there is none."""
    dist = torch.distributed
    given = (group,) if _world(group) > 1 else ()
    if not _sharded(t):
        return given
    mesh, split = t.device_mesh, []
    for d, p in enumerate(t.placements):
        if mesh.size(d) == 1 or p.is_replicate():
            continue
        if not (p.is_shard() or hasattr(p, "split_factor")):      # (a shard of a shard says no to is_shard)
            raise ValueError(f"{name} expects gradients that are reduced over their mesh, got the placements {t.placements}")
        split.append(d)
    if group is None:
        return tuple(mesh.get_group(d) for d in split)
    here = mesh.get_coordinate()
    ranks = mesh.mesh[tuple(slice(None) if d in split else here[d] for d in range(mesh.ndim))].flatten().tolist()
    if sorted(ranks) != sorted(dist.get_process_group_ranks(group)):
        raise ValueError(f"{name} over the ranks {dist.get_process_group_ranks(group)} expects tensors whose parts lie on these, got one with the "
                         f"placements {t.placements} whose parts lie on {ranks}; without a group the norm is taken over each one's mesh")
    return given


def _reduced(total: torch.Tensor, inf: bool, group) -> torch.Tensor:
    dist = torch.distributed
    if inf:      # by their bits: the largest of numbers, and a NaN above them all
        total = total.abs()
        dist.all_reduce(total.view(torch.int64), op=dist.ReduceOp.MAX, group=group)
    else:
        dist.all_reduce(total, op=dist.ReduceOp.SUM, group=group)
    return total


def _world(group) -> int:
    dist = torch.distributed
    return dist.get_world_size(group) if group is not None and dist.is_initialized() else 1


def _over(name: str, total: Optional[torch.Tensor], inf: bool, group) -> torch.Tensor:
    """The total over the ranks of ``group``.  A rank without tensors (None) takes part with nothing, so that the others do not wait for it,
    and learns whether any has one."""
    if total is None:
        own = torch.zeros(2, dtype=torch.float64, device="cuda" if torch.cuda.is_available() else "cpu")
    else:
        own = torch.stack([total, torch.ones_like(total)])
    got = _reduced(own, inf, group)
    if total is None and float(got[1]) == 0.0:
        raise ValueError(f"{name} over ranks expects a tensor on each, or on one of them at least: none has any")
    return got[0]


def _norm(name: str, tensors: Sequence[torch.Tensor], inf: bool, group):
    """(total, norm), over the ranks of ``group`` and of the tensors' meshes too."""
    if not tensors:
        total = _over(name, None, inf, group)
        return total, (total if inf else total.sqrt()).float()
    host = L._autograd_module or L.autograd()
    got = host.grad_norm(tensors, inf)
    if got is not None:
        total, norm = got
        if _world(group) > 1:
            total = _over(name, total, inf, group)
            norm = (total if inf else total.sqrt()).float()
        return total, norm
    parts: dict = {}           # the groups' names -> (groups, tensors whose parts lie on them)
    for t in tensors:
        groups = _holders(name, t, group)
        parts.setdefault(tuple(g.group_name for g in groups), (groups, []))[1].append(_local(t))
    totals = []
    for _, local in parts.values():
        got = host.grad_norm(local, inf)
        if got is None:
            _refuse(name, tensors)
        totals.append(got[0])
    for i, (groups, _) in enumerate(parts.values()):
        for g in groups:
            totals[i] = _over(name, totals[i], inf, g) if g is group else _reduced(totals[i], inf, g)
    total = totals[0]
    if len(totals) > 1:
        total = torch.stack(totals).amax() if inf else torch.stack(totals).sum()
    return total, (total if inf else total.sqrt()).float()


@L.traced("grad_norm")
def grad_norm(tensors: Iterable[torch.Tensor], norm_type: float = 2.0, group=None) -> torch.Tensor:
    """fp32 scalar: the 2-norm (or the largest magnitude, ``norm_type`` inf) of all tensors together, of DTensors as whole ones:
    over the ranks of their meshes that they are sharded over (replicas count once; all ranks list the same ones).  ``group``: over
    the ranks of it, each of which holds a part of everything, or nothing (such a rank waits for the answer); DTensors have to
    be sharded over just these."""
    inf = _kind(norm_type)
    tensors = _list(tensors)
    if not tensors and _world(group) == 1:
        return torch.zeros(())
    return _norm("grad_norm", tensors, inf, group)[1]


@L.traced("clip_grads")
def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0, out: Optional[Sequence[torch.Tensor]] = None,
               group=None, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the tensors (which do not overlap) to a common norm of at most ``max_norm``, in place or into ``out`` (of the same
    shapes and types: others, or the gradient itself in its own place); returns the norm before, an fp32 scalar.  Where nothing is clipped, tensors scaled in place are not
    written.  DTensors and ``group``: as ``grad_norm`` takes them; ``out`` is sharded like ``grads``, and a norm over ranks needs the call
    on all of them.  ``error_if_nonfinite`` waits for the norm and raises before anything is scaled."""
    inf, max_norm = _kind(norm_type), float(max_norm)
    grads, outs = _list(grads), [] if out is None else _list(out)
    if not grads and _world(group) == 1:
        return torch.zeros(())
    if out is not None and len(outs) != len(grads):
        raise ValueError("clip_grads expects out like grads: as many tensors, of their shapes and types")
    total = None
    if error_if_nonfinite or _world(group) > 1:
        total, norm = _norm("clip_grads", grads, inf, group)
        if error_if_nonfinite and not math.isfinite(float(total)):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is non-finite, so it cannot "
                               "be clipped. To disable this error and scale the gradients by the non-finite norm anyway, set "
                               "`error_if_nonfinite=False`")
        if not grads:
            return norm
    host = L._autograd_module or L.autograd()
    got = host.clip_grads(grads, outs, max_norm, inf, total)
    if got is None:
        whole = [_sharded(t) for t in (*grads, *outs)]
        if any(whole):
            for g, o in zip(grads, outs):
                if _sharded(g) != _sharded(o) or (_sharded(g) and (g.placements != o.placements or g.device_mesh != o.device_mesh)):
                    raise ValueError("clip_grads expects out like grads: as many tensors, of their shapes and types, sharded like them")
            if total is None:
                total, _ = _norm("clip_grads", grads, inf, group)
        got = host.clip_grads([_local(g) for g in grads], [_local(o) for o in outs], max_norm, inf, total)
        if got is None:
            _refuse("clip_grads", grads, outs)
        torch.autograd.graph.increment_version([t for t in outs or grads if _sharded(t) and not t.is_inference()])
    return got


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, group=None) -> torch.Tensor:
    """``clip_grads`` of the gradients that the parameters have, DTensors among them (their norm is taken over the mesh)."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_grads([p.grad for p in parameters if p.grad is not None], max_norm, norm_type, None, group, error_if_nonfinite)
