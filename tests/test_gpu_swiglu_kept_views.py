"""Kept SwiGLU of rows cut out of another buffer: one row, whose stride says nothing, and pointers off 16 bytes.  Bit for bit the
call on a copy."""
import pytest
import torch

from alto_b200.swiglu import swiglu

pytestmark = pytest.mark.gpu


def _buffer(rows, cols, seed=0):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


def _views():
    yield _buffer(4, 133)[:1, :128]                        # one row of an odd pitch
    yield _buffer(4, 132)[2:3, :128]
    yield _buffer(4, 133)[1:2, :128]                       # and off 16 bytes
    yield _buffer(128, 3)[:, :1].t()                       # a transposed column, copied
    yield _buffer(128, 1).t()                              # a transposed column that is contiguous, with a stride of 1
    yield _buffer(1, 5 * 128 + 3)[0, 3:].view(5, 128)      # several contiguous rows off 16 bytes
    yield _buffer(9, 192)[:, 64:]


@pytest.mark.parametrize("checkpoint", ["e4m3", "e5m2", None])
def test_rows_of_another_buffer(checkpoint):
    for i, h in enumerate(_views()):
        rows, hidden = h.shape[0], h.shape[1] // 2
        dys = (_buffer(rows, hidden, 1), _buffer(1, rows * hidden + 1, 2)[0, 1:].view(rows, hidden))
        for dy in dys:
            leaf, copy = h.detach().requires_grad_(True), h.clone(memory_format=torch.contiguous_format).view(-1).view(rows, 2 * hidden).requires_grad_(True)
            y, want = swiglu(leaf, checkpoint=checkpoint), swiglu(copy, checkpoint=checkpoint)
            assert torch.equal(y, want), i
            (dh,), (want_dh,) = torch.autograd.grad(y, leaf, dy), torch.autograd.grad(want, copy, dy.clone())
            assert torch.equal(dh, want_dh), i
