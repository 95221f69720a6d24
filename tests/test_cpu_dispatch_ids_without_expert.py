"""Ids outside [0, num_experts) in the expert-parallel dispatcher: slots without an expert, on any number of ranks.  Two gloo ranks
on CPU, and one; against a dense computation that leaves those slots out."""
import pytest
import torch

from alto_b200 import distributed as D
from tests.test_cpu_distributed import _experts, _gather_rows_cpu, _spawn


def _ids(T, k, num_experts, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, num_experts, (T, k), generator=g)
    ids[3], ids[7, 0], ids[9, -1], ids[11, 0] = -1, num_experts, -2 ** 40, num_experts + 5
    return ids


def _check(T, k, num_experts, seed, rank, world, ids):
    g = torch.Generator().manual_seed(100 + seed)
    W = torch.randn(num_experts, 16, 24, generator=torch.Generator().manual_seed(7), dtype=torch.float64)
    x = torch.randn(T, 16, generator=g, dtype=torch.float64, requires_grad=True)
    scores = torch.rand(T, k, generator=g, dtype=torch.float64).requires_grad_(True)
    d = D.ExpertParallelDispatcher(num_experts)
    x_local, offs, st = d.dispatch(x, ids)
    E = num_experts // world
    assert offs.numel() == E and x_local.shape[0] == int(offs[-1])
    out = d.combine(_experts(x_local, offs, W[rank * E:(rank + 1) * E]), st, scores)
    xr, sr = x.detach().clone().requires_grad_(True), scores.detach().clone().requires_grad_(True)
    there = ((ids >= 0) & (ids < num_experts)).double()
    safe = ids.clamp(0, num_experts - 1)
    ref = sum((sr * there)[:, j:j + 1] * torch.einsum("td,tdo->to", xr, W[safe[:, j]]) for j in range(k))
    assert torch.allclose(out, ref, rtol=1e-12, atol=1e-12)
    up = torch.randn(T, 24, generator=g, dtype=torch.float64)
    (out * up).sum().backward()
    (ref * up).sum().backward()
    assert torch.allclose(x.grad, xr.grad, rtol=1e-12, atol=1e-12) and torch.allclose(scores.grad, sr.grad, rtol=1e-12, atol=1e-12)


def _worker(rank, world, num_experts, T, k):
    _check(T, k, num_experts, rank, rank, world, _ids(T, k, num_experts, rank))
    # a rank without a single routed row
    _check(T, k, num_experts, rank, rank, world, _ids(T, k, num_experts, rank) if rank == 0 else torch.full((T, k), -1))


@pytest.mark.parametrize("num_experts, k", [(4, 2), (8, 3)])
def test_two_ranks(num_experts, k):
    _spawn(_worker, num_experts, 40, k)


def test_one_rank(monkeypatch):
    monkeypatch.setattr(D.L, "gather_rows", _gather_rows_cpu)
    _check(40, 2, 4, 0, 0, 1, _ids(40, 2, 4, 0))
    _check(12, 2, 4, 0, 0, 1, torch.full((12, 2), 4))
