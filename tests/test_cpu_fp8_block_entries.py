"""What the C entry points of the FP8 block operators and of clipping answer to arguments that they do not take: a status, before
any launch.  And the reduction of a norm over ranks, as two gloo ranks."""
import ctypes as C
import math
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from alto_b200 import _lib as L
from alto_b200 import grad_clip as GC

P = 1 << 20            # never read: every call ends before a launch
SCALE = L.Fp8BlockScale(P, 1, 1, 0, 0, 7)


def quant(**kw):
    a = dict(x=P, rows=4, cols=32, ld=32, offs=None, row_codes=P, row_scales=P, col_codes=None, col_scales=None, ld_col=0, dtype=L.DT_BF16, format=2,
             experts=0)
    a.update(kw)
    return L.Fp8BlockQuantArgs(*(a[n] for n, _ in L.Fp8BlockQuantArgs._fields_))


@pytest.mark.parametrize("change", [dict(cols=0), dict(cols=24), dict(rows=-1), dict(ld=16), dict(x=None), dict(x=P + 2), dict(row_codes=P + 8),
                                    dict(ld=36), dict(dtype=7), dict(format=1), dict(row_codes=None), dict(row_scales=None),
                                    dict(col_codes=P, col_scales=P, ld_col=64), dict(col_codes=P, col_scales=None, ld_col=128),
                                    dict(rows=1 << 30), dict(col_codes=P, col_scales=P, ld_col=128, offs=P, experts=2)], ids=str)
def test_quantizer(change):
    assert L.lib().altob200_fp8_block_quantize(quant(**change), None) < 0


def test_nothing_to_quantise():
    assert L.lib().altob200_fp8_block_quantize(quant(rows=0), None) == 0
    assert L.lib().altob200_fp8_block_quantize(None, None) == L.E_SHAPE


@pytest.mark.parametrize("change", [dict(dtype=7), dict(format=0), dict(matrices=-1), dict(rows=0), dict(rows=24), dict(cols=8), dict(cols=24), dict(ld=8),
                                    dict(ld=36), dict(stride=36), dict(x=None), dict(x=P + 4), dict(codes=P + 8), dict(turned=P + 8),
                                    dict(codes=None, turned=None), dict(scales=None), dict(matrices=70000), dict(rows=128 * 65536)], ids=str)
def test_squares(change):
    a = dict(x=P, dtype=L.DT_BF16, format=2, matrices=1, rows=32, cols=32, ld=32, stride=32 * 32, codes=P, turned=P, scales=P)
    a.update(change)
    assert L.lib().altob200_fp8_block_quantize_squares(*a.values(), None) < 0


@pytest.mark.parametrize("change", [dict(format=0), dict(cols=4), dict(rows=-1), dict(codes=None), dict(codes=P + 4), dict(out=None), dict(out=P + 4),
                                    dict(dtype=9), dict(scale=L.Fp8BlockScale(None, 1, 1, 0, 0, 7)), dict(scale=L.Fp8BlockScale(P, 1, 1, 0, 3, 7)),
                                    dict(scale=None)], ids=lambda d: next(iter(d)))
def test_values(change):
    a = dict(codes=P, format=2, rows=4, cols=32, scale=SCALE, dtype=L.DT_F32, out=P)
    a.update(change)
    assert L.lib().altob200_fp8_block_dequantize(*a.values(), None) < 0


@pytest.mark.parametrize("change", [dict(M=-1), dict(N=0), dict(N=24), dict(K=24), dict(K=-16), dict(ldd=16), dict(format=0), dict(mode=3), dict(mode=1),
                                    dict(mode=1, offs=P, experts=0), dict(a_dtype=5), dict(mode=2, offs=P, experts=1, a_dtype=L.DT_BF16),
                                    dict(mode=2, offs=P, experts=1, k_rows=300), dict(out_dtype=9), dict(a=P + 8), dict(b=P + 8), dict(d=P + 8),
                                    dict(ldd=36, out_dtype=L.DT_BF16), dict(a=None), dict(b=None), dict(d=None), dict(a_dtype=L.DT_BF16, lda=16),
                                    dict(a_dtype=L.DT_F32, lda=34), dict(M=1 << 30), dict(K=1 << 30), dict(mode=1, offs=P, experts=40000),
                                    dict(sa=L.Fp8BlockScale(P, 1, 1, 0, 5, 7)), dict(sa=L.Fp8BlockScale()), dict(sb=L.Fp8BlockScale())], ids=str)
def test_product(change):
    a = dict(M=4, N=32, K=32, lda=32, ldd=32, k_rows=0, a=P, b=P, sa=SCALE, sb=SCALE, offs=None, d=P, mode=0, experts=0, format=2, a_dtype=-1,
             out_dtype=L.DT_F32, b_ready=0)
    a.update(change)
    assert L.lib().altob200_fp8_block_gemm(L.Fp8BlockGemmArgs(*a.values()), None) < 0


def test_no_rows():
    a = L.Fp8BlockGemmArgs(0, 32, 32, 32, 32, 0, None, P, L.Fp8BlockScale(), SCALE, None, None, 0, 0, 2, L.DT_F32, L.DT_F32, 0)
    assert L.lib().altob200_fp8_block_gemm(a, None) == 0 and L.lib().altob200_fp8_block_gemm(None, None) == L.E_SHAPE


def grads(pointers, sizes, dtypes, outs=None):
    n = len(sizes)
    keep = ((C.c_void_p * n)(*pointers), (C.c_void_p * n)(*(outs or pointers)), (C.c_int64 * n)(*sizes), (C.c_int32 * n)(*dtypes))
    return L.GradList(*(C.cast(k, C.c_void_p) for k in keep), n), keep


@pytest.mark.parametrize("pointers,sizes,dtypes,outs", [([None], [3], [L.DT_F32], None), ([P], [-1], [L.DT_F32], None), ([P], [3], [7], None),
                                                        ([P + 2], [3], [L.DT_F32], None), ([P, P + 1], [3, 3], [L.DT_BF16] * 2, None),
                                                        ([P], [3], [L.DT_F32], [None])], ids=str)
def test_lists(pointers, sizes, dtypes, outs):
    l, keep = grads(pointers, sizes, dtypes, outs)
    assert L.lib().altob200_clip_grads(l, 0, 1.0, None, P, P, None) < 0
    assert L.lib().altob200_grad_norm(l, 0, P, P, P, None) < 0
    good, keep2 = grads([P], [3], [L.DT_F32])
    assert L.lib().altob200_grad_norm(good, 0, None, P, P, None) < 0 and L.lib().altob200_clip_grads(good, 0, 1.0, None, P + 4, P, None) < 0
    assert L.lib().altob200_grad_norm(None, 0, P, P, P, None) < 0


@pytest.mark.parametrize("src,counts", [(None, P), (P, None), (P + 8, P), (P, P + 2)], ids=str)
def test_selftest_of_the_copies(src, counts):
    assert L.lib().altob200_selftest_drain(src, counts, None) < 0


def _norms(rank, port):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        group = dist.group.WORLD
        assert GC._world(group) == 2 and GC._world(None) == 1
        assert float(GC._reduced(torch.tensor(3.0 + rank, dtype=torch.float64), False, group)) == 7.0
        assert float(GC._reduced(torch.tensor(3.0 + rank, dtype=torch.float64), True, group)) == 4.0
        for bad in (math.nan, -math.nan, math.inf):          # on either rank
            for where in (0, 1):
                got = float(GC._reduced(torch.tensor(bad if rank == where else 5.0, dtype=torch.float64), True, group))
                assert math.isnan(got) if math.isnan(bad) else got == math.inf
        for call in (lambda: GC.grad_norm([], group=group), lambda: GC.clip_grads([], 1.0, group=group)):
            with pytest.raises(ValueError, match="a tensor on each"):
                call()
    finally:
        dist.destroy_process_group()


def test_norm_over_ranks():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_norms, args=(port,), nprocs=2, join=True)
