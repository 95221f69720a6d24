"""Routing of tokens to experts in front of the grouped GEMMs.

    ids, weights = route_experts(logits, top_k, ...)      the chosen experts and their weights, differentiable in logits
    plan = expert_plan(ids, num_experts)                  rows of the expert-major, padded token buffer

``distributed.ExpertParallelDispatcher`` takes ``ids`` in ``dispatch`` and ``weights`` as the scores of ``combine``; on one
rank it builds its row plan with ``expert_plan``.  ``plan.token`` is the index that gathers tokens into the buffer
(``-1``: a padding row of zeros), ``plan.offs`` what the functions of ``alto_b200.grouped`` take as ``offs``.

The reference leaves routing and dispatch to its TorchTitan fork (alto/modifiers/lpt/base.py:194-201)."""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib as L

__all__ = ["route_experts", "expert_plan", "ExpertPlan"]

ALIGN_SIZE_M = 128
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS, MAX_PLAN_EXPERTS = 512, 16, 32, 1024
_SCORES = {"softmax": 0, "sigmoid": 1}


class ExpertPlan(NamedTuple):
    """Rows of the padded buffer, int32.  ``token`` / ``position`` [rows]: token and routed slot (t * k + j) of a row, -1 in
    padding; ``slot`` [tokens * k]: row of a routed slot, -1 where it has none; ``offs`` [experts]: ends of the padded
    runs; ``counts`` [experts]: rows of the runs without padding."""
    token: torch.Tensor
    position: torch.Tensor
    slot: torch.Tensor
    offs: torch.Tensor
    counts: torch.Tensor


def _rows(t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    elif t.is_contiguous() and t.shape[0] > 1 and t.shape[1] > 1:      # the usual case, with the fewest questions
        return t
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:      # one expert or one token: strides that say nothing
        t = t.as_strided(t.shape, (t.shape[1], 1))
    return t


def _forward(logits, params, bias):
    return L.route_forward(_rows(logits), params, bias, None if logits.dim() == 2 else logits.shape[:-1])


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, params, bias):
        ids, weights = _forward(logits, params, bias)
        ctx.save_for_backward(logits, ids)
        ctx.params = params
        ctx.set_materialize_grads(False)      # no zeros in the place of a gradient of ids
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    @L.once_differentiable
    def backward(ctx, _, grad):
        if grad is None:
            return None, None, None
        logits, ids = ctx.saved_tensors
        g = L.route_backward(_rows(logits), ctx.params, ids, grad if grad.is_contiguous() else grad.contiguous())
        return (g if logits.dim() == 2 else g.view(logits.shape)), None, None


@L.traced("route_experts")
def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
                  num_groups: int = 1, groups_kept: int = 1, group_top: int = 1, renormalize: bool = True,
                  scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(ids int32 [..., top_k], weights fp32 [..., top_k]) of logits [..., experts] (bf16 or fp32).

    The ``top_k`` experts with the largest ``score`` ("softmax" over the experts or "sigmoid") plus ``bias`` (fp32
    [experts], for balance: it moves the choice, not the weights, and gets no gradient) are chosen, largest first, the
    lowest index first among equals.  Keys are compared as if they had 64 bits.  With ``num_groups`` > 1 only experts of the
    ``groups_kept`` groups of neighbours whose best ``group_top`` (1 or 2) keys have the largest sum can be chosen.

    The weights are the chosen experts' scores, divided by their sum with ``renormalize``, times ``scale``.  A token whose
    chosen scores are all zero (every logit -inf) gets zero weights.  Differentiable in ``logits``.  At most 512 experts, 16 of
    them chosen, 32 groups."""
    if not logits.is_cuda or (bias is not None and not bias.is_cuda):
        raise RuntimeError("route_experts runs on CUDA tensors only (no CPU fallback)")
    if logits.dim() < 1 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"route_experts expects bfloat16 or float32 logits [..., experts], got {logits.dtype}, {tuple(logits.shape)}")
    experts = logits.shape[-1]
    if score not in _SCORES:
        raise ValueError(f"unsupported score {score!r}; supported: {sorted(_SCORES)}")
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"route_experts takes 1 to {MAX_EXPERTS} experts, got {experts}")
    if not 1 <= num_groups <= MAX_GROUPS or experts % num_groups != 0:
        raise ValueError(f"{experts} experts do not split into {num_groups} groups (at most {MAX_GROUPS})")
    if not 1 <= groups_kept <= num_groups or group_top not in (1, 2):
        raise ValueError(f"groups_kept {groups_kept} of {num_groups} groups, group_top {group_top} (1 or 2)")
    if not 1 <= top_k <= min(MAX_TOP_K, groups_kept * (experts // num_groups)):
        raise ValueError(f"top_k {top_k}: at most {MAX_TOP_K}, and at most the {groups_kept * (experts // num_groups)} experts to choose from")
    if bias is not None:
        if bias.shape != (experts,) or bias.device != logits.device:
            raise ValueError(f"route_experts expects a bias of [{experts}] on {logits.device}, got {tuple(bias.shape)} on {bias.device}")
        bias = bias.detach().float().contiguous()
    params = L.RouteParams(L._dt(logits.dtype), experts, top_k, _SCORES[score], num_groups, groups_kept, group_top,
                           1 if renormalize else 0, scale)
    if logits.requires_grad and torch.is_grad_enabled() or L.forward_mode():
        return _Route.apply(logits, params, bias)
    return _forward(logits, params, bias)


@L.traced("expert_plan")
def expert_plan(expert_ids: torch.Tensor, num_experts: int, align: int = ALIGN_SIZE_M, rows: Optional[int] = None) -> ExpertPlan:
    """The row plan of the buffer in which every expert's tokens are neighbours: routed slots in their order within an
    expert, every run padded to a multiple of ``align`` rows (an expert without tokens gets one run of padding).

    ``expert_ids``: int32 or int64 [..., k]; a number outside [0, num_experts) is a slot without an expert.  ``rows``:
    rows of the buffer; by default what holds every run however the tokens are routed,
    ``(tokens * k + num_experts * align) // align * align``, so that nothing waits for the counts.  Slots whose row does not
    fit into ``rows`` are dropped (``offs`` are the runs' ends all the same; the grouped GEMMs cut them off at the buffer's
    end).  For the grouped GEMMs ``align`` is a multiple of 128.  At most 1024 experts."""
    if not expert_ids.is_cuda:
        raise RuntimeError("expert_plan runs on CUDA tensors only (no CPU fallback)")
    if expert_ids.dtype not in (torch.int32, torch.int64) or expert_ids.dim() < 1:
        raise TypeError(f"expert_plan expects int32 or int64 ids [..., k], got {expert_ids.dtype}, {tuple(expert_ids.shape)}")
    if not 1 <= num_experts <= MAX_PLAN_EXPERTS:
        raise ValueError(f"expert_plan takes 1 to {MAX_PLAN_EXPERTS} experts, got {num_experts}")
    if align < 1 or expert_ids.shape[-1] < 1:
        raise ValueError(f"expert_plan expects align >= 1 and k >= 1, got {align} and {expert_ids.shape[-1]}")
    k, slots = expert_ids.shape[-1], expert_ids.numel()
    if slots + num_experts * align >= 2 ** 31 - 1 or (rows is not None and not 0 <= rows < 2 ** 31 - 1):
        raise ValueError(f"expert_plan: {slots} slots, {num_experts} experts x {align}, {rows} rows do not fit 32-bit row numbers")
    if rows is None:
        rows = (slots + num_experts * align) // align * align
    return ExpertPlan(*L.expert_plan(expert_ids.contiguous(), slots // k, k, num_experts, align, rows))
