"""The norm's step through autograd at a size where the host is what counts, and what the graph around it does."""
import time

import pytest
import torch
import torch.utils.checkpoint

from alto_b200 import norm

pytestmark = pytest.mark.gpu


def _time(call, n=300):
    best = float("inf")
    for _ in range(6):
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(n):
            call()
        torch.cuda.synchronize()
        best = min(best, time.perf_counter() - start)
    return best / n * 1e6


def test_a_small_step_takes_no_longer_than_tensor_operations():
    g = torch.Generator(device="cuda").manual_seed(0)
    x, dy = (torch.randn(1023, 1537, generator=g, device="cuda") for _ in range(2))
    w = torch.ones(1537, device="cuda")
    leaf, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    def plain():      # nothing that autograd would keep, no graph
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
        xhat = x * rstd
        gw = dy * w
        return xhat * w, rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True)), (dy * xhat).sum(0)

    def step():
        y = norm.rms_norm(leaf, wl)
        return y, *torch.autograd.grad(y, (leaf, wl), dy)
    took = _time(step), _time(plain)
    assert took[0] <= took[1], took


def test_second_derivatives_are_refused_whatever_is_differentiated():
    x, w = torch.randn(8, 64, device="cuda"), torch.ones(64, device="cuda")
    for which in range(3):
        leaf, wl, res = (t.clone().requires_grad_(True) for t in (x, w, x))
        y, r = norm.rms_norm(leaf, wl, residual=res)
        grads = torch.autograd.grad(y, (leaf, wl, res), torch.ones_like(y), create_graph=True)
        with pytest.raises(RuntimeError, match="rms_norm"):
            grads[which].sum().backward()
    # through the stream alone there is one: the gradient is the upstream gradient itself
    up = torch.randn(8, 64, device="cuda", requires_grad=True)
    _, r = norm.rms_norm(leaf, wl, residual=res)
    (gx,) = torch.autograd.grad(r, leaf, up, create_graph=True)
    (gx * 3).sum().backward()
    assert (up.grad == 3).all()


def test_a_graph_is_freed_by_its_backward_pass_and_may_be_kept():
    leaf, w = torch.randn(8, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda", requires_grad=True)
    y = norm.rms_norm(leaf, w)
    first = torch.autograd.grad(y, (leaf, w), torch.ones_like(y), retain_graph=True)
    second = torch.autograd.grad(y, (leaf, w), torch.ones_like(y))
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaf, torch.ones_like(y))
    # a saved operand that was written to
    leaf2 = leaf.detach().clone().requires_grad_(True)
    x = leaf2 * 1.0
    y = norm.rms_norm(x, w)
    x += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    # rematerialised under a checkpoint
    y = torch.utils.checkpoint.checkpoint(lambda t: norm.rms_norm(t, w), leaf, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(y, leaf, torch.ones_like(y))[0], first[0])


def test_gradients_of_nothing_that_asks_for_one():
    x, w = torch.randn(8, 64, device="cuda"), torch.ones(64, device="cuda")
    res = x.clone().requires_grad_(True)
    y, r = norm.rms_norm(x, w, residual=res)
    (g,) = torch.autograd.grad((y, r), res, (torch.ones_like(y), torch.ones_like(r)))
    assert g.shape == res.shape
    with torch.no_grad():
        assert not norm.rms_norm(res, w).requires_grad
    assert not norm.rms_norm(x, w).requires_grad and norm.rms_norm(res, w).requires_grad



def test_a_refused_call_raises_the_package_error():
    from alto_b200 import _lib as L
    x = torch.zeros(1, device="cuda", dtype=torch.bfloat16).expand(2 ** 31, 1)      # more rows than the kernels count
    with pytest.raises(L.Altob200Error, match="altob200_rms_norm_forward") as e:
        norm.rms_norm(x, x[0])
    assert e.value.status == L.E_LIMIT


def test_one_tensor_as_rows_and_residual():
    x, w = torch.randn(8, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda")
    copy = x.detach().clone().requires_grad_(True)
    up = torch.randn(8, 64, device="cuda")
    (once,) = torch.autograd.grad(norm.rms_norm(x, w, residual=copy)[0], x, up)
    (twice,) = torch.autograd.grad(norm.rms_norm(x, w, residual=x)[0], x, up)
    assert torch.equal(twice, once * 2)
    x.grad = None
    norm.rms_norm(x, w, residual=x)[0].backward(up)
    norm.rms_norm(x, w, residual=copy)[0].backward(up)
    assert torch.allclose(x.grad, once * 3, rtol=2.0 ** -22) and torch.equal(copy.grad, once)


def test_inference_mode_and_hooks_around_saved_tensors():
    x, w = torch.randn(4, 8, 64, device="cuda"), torch.ones(64, device="cuda")
    want = norm.rms_norm(x, w, residual=x)
    with torch.inference_mode():
        got = norm.rms_norm(x, w, residual=x)
        inside = norm.rms_norm(got[1], w)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(inside, norm.rms_norm(want[1], w))
    leaf, seen = x.clone().requires_grad_(True), []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t.cpu(), lambda t: t.cuda()):
        y = norm.rms_norm(leaf, w)
    (g,) = torch.autograd.grad(y, leaf, x)
    leaf2 = x.clone().requires_grad_(True)
    assert len(seen) == 2 and torch.equal(g, torch.autograd.grad(norm.rms_norm(leaf2, w), leaf2, x)[0])


def test_steps_from_several_threads():
    import threading
    x, w, up = torch.randn(200, 512, device="cuda"), torch.ones(512, device="cuda"), torch.randn(200, 512, device="cuda")

    def step():
        leaf, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        return torch.autograd.grad(norm.rms_norm(leaf, wl), (leaf, wl), up)
    want, got = step(), {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got[i] = step()
        torch.cuda.synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert len(got) == 4 and all(torch.equal(a, b) for g in got.values() for a, b in zip(g, want))
