"""The FP8 format with one fp32 scale for each block of 128, restated with elementary CPU operations, and how far sums may be off."""
from __future__ import annotations

import torch

BLOCK = 128
TOP = {"e4m3": 448.0, "e5m2": 57344.0}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def blocks(n):
    return -(-n // BLOCK)


def quantize(t, fmt, dim):
    """(codes, scales, values in fp64) of a CPU matrix; ``dim``: -1 blocks of a row, -2 blocks of a column, None squares."""
    t = t.detach().float()
    rows, cols = t.shape
    br, bc = (1 if dim == -1 else BLOCK), (1 if dim == -2 else BLOCK)
    nr, nc = -(-rows // br), -(-cols // bc)
    full = torch.zeros(nr * br, nc * bc)
    full[:rows, :cols] = t
    tiles = full.view(nr, br, nc, bc)
    top = torch.tensor(TOP[fmt])
    largest = tiles.abs().amax(3).amax(1)
    scales = torch.where(torch.isnan(largest), largest, largest.clamp_min(1e-12)) / top
    q = tiles / scales[:, None, :, None]
    codes = torch.where(torch.isnan(q), q, q.clamp(-TOP[fmt], TOP[fmt])).to(F8[fmt])
    values = codes.double() * scales.double()[:, None, :, None]
    return codes.view(nr * br, nc * bc)[:rows, :cols], scales, values.view(nr * br, nc * bc)[:rows, :cols]


def product_bound(a, b, out_dtype):
    """(a b^T, how far each element may be off): every product of codes is exact, and a sum of K of them in fp32, in whatever
    order and rounded or cut off, takes at most 128 additions in a block and one product and addition for each block, each
    off by 2^-23 of a partial sum that is no larger than the sum of magnitudes; the scales' product is rounded too.  bf16
    adds half a step of the result, 2^-8."""
    exact, size = a @ b.T, a.abs() @ b.abs().T
    bound = size * (BLOCK + 3 * blocks(a.shape[1])) * 2.0 ** -23
    if out_dtype == torch.bfloat16:
        bound = bound + (exact.abs() + bound) * 2.0 ** -8
    return exact, bound


def assert_within(got, exact, bound, what=""):
    off = (got.detach().cpu().double() - exact).abs() - bound
    worst = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or float(off.flatten()[worst]) <= 0.0, (
        f"{what}: element {worst} is {float(got.detach().cpu().double().flatten()[worst])}, expected {float(exact.flatten()[worst])} "
        f"within {float(bound.flatten()[worst])}")


def numbers(shape, dtype, seed, std=1.0, loud=True):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(shape, generator=g) * std
    if loud and t.numel():
        t = t * torch.where(torch.rand(shape[-1], generator=g) < 0.05, 30.0, 1.0)
    return t.to(dtype)


def runs(counts):
    ends, at = [], 0
    for c in counts:
        at += c
        ends.append(at)
    return torch.tensor(ends, dtype=torch.int32)
