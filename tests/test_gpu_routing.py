"""Routing and the row plan against plain forms: the choice exactly, weights and gradients in 64 bits.

Tolerances: a weight is a ratio of exponentials whose arguments are off by 2^-24 of themselves (at most 32 here), each
exponential by two steps, sums by their 16 or 512 / 32 + 5 terms, the quotient and the scale by half a step each: below
(32 + 4 + 21 + 4) 2^-24 < 2^-18.  A gradient is the product of such weights with differences of upstream gradients."""
import numpy as np
import pytest
import torch

from alto_b200 import routing

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
W = 2.0 ** -18


def route64(logits, k, score="softmax", bias=None, num_groups=1, groups_kept=1, group_top=1, renormalize=True, scale=1.0):
    """(ids, weights, scores) by definition, in 64 bits."""
    l = logits.double().cpu()
    s = torch.sigmoid(l) if score == "sigmoid" else torch.nan_to_num(torch.softmax(l, -1)) if torch.isinf(l).all(-1).any() else torch.softmax(l, -1)
    if bias is None and (group_top == 1 or groups_kept == num_groups):
        key = l.clone()
    else:
        key = s + (0 if bias is None else bias.double().cpu())
    size = l.shape[-1] // num_groups
    if groups_kept < num_groups:
        of = torch.sort(key.unflatten(-1, (num_groups, size)), dim=-1, descending=True).values[..., :group_top].sum(-1)
        order = torch.sort(of, dim=-1, descending=True, stable=True).indices
        drop = torch.ones_like(of, dtype=torch.bool).scatter(-1, order[..., :groups_kept], False)
        key = torch.where(drop.repeat_interleave(size, -1), torch.full_like(key, -torch.inf), key)
        # of kept groups, experts of -inf stay in front of those that cannot be chosen
        rank = drop.repeat_interleave(size, -1).double()
    else:
        rank = torch.zeros_like(key)
    first = torch.sort(key, dim=-1, descending=True, stable=True).indices
    again = torch.sort(rank.gather(-1, first), dim=-1, stable=True).indices
    ids = first.gather(-1, again)[..., :k]
    chosen = s.gather(-1, ids)
    total = chosen.sum(-1, keepdim=True) if renormalize else torch.ones_like(chosen[..., :1])
    weights = torch.where(total > 0, chosen / total, torch.zeros_like(chosen)) * scale
    return ids, weights, s


def grad64(ids, s, g, score, renormalize, scale):
    g = g.double().cpu() * scale
    chosen = s.gather(-1, ids)
    if renormalize:
        total = chosen.sum(-1, keepdim=True)
        q = torch.where(total > 0, chosen / total, torch.zeros_like(chosen))
        slope = q * (1 - chosen) if score == "sigmoid" else q
        d = slope * (g - (g * q).sum(-1, keepdim=True))
        size = slope * (g.abs() + (g * q).abs().sum(-1, keepdim=True))
        return torch.zeros_like(s).scatter(-1, ids, d), torch.zeros_like(s).scatter(-1, ids, size)
    if score == "sigmoid":
        d = chosen * (1 - chosen) * g
        return torch.zeros_like(s).scatter(-1, ids, d), torch.zeros_like(s).scatter(-1, ids, d.abs())
    up = torch.zeros_like(s).scatter(-1, ids, g)
    dot, size = (up * s).sum(-1, keepdim=True), (up * s).abs().sum(-1, keepdim=True)
    return s * (up - dot), s * (up.abs() + size)


def _logits(tokens, experts, dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(tokens, experts, generator=g, device="cuda") * std).to(dtype)


def _check(logits, k, **options):
    bias = options.get("bias")
    leaf = logits.clone().requires_grad_(True)
    ids, weights = routing.route_experts(leaf, k, **options)
    want_ids, want_w, s = route64(logits, k, **options)
    assert ids.dtype == torch.int32 and weights.dtype == torch.float32
    assert torch.equal(ids.cpu().long(), want_ids)
    w = weights.detach().cpu().double()
    assert ((w - want_w).abs() <= want_w.abs() * W + 1e-37).all()
    g = torch.Generator(device="cuda").manual_seed(9)
    up = torch.randn(weights.shape, generator=g, device="cuda")
    (dl,) = torch.autograd.grad(weights, leaf, up)
    assert dl.dtype == logits.dtype and dl.shape == logits.shape
    score, renorm = options.get("score", "softmax"), options.get("renormalize", True)
    want, size = grad64(want_ids, s, up, score, renorm, options.get("scale", 1.0))
    assert ((dl.cpu().double() - want).abs() <= want.abs() * HALF[dl.dtype] + size * 4 * W + 1e-37).all()
    with torch.no_grad():
        again = routing.route_experts(logits, k, **options)
    assert torch.equal(again[0], ids) and torch.equal(again[1], weights.detach())
    return ids, weights


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens, experts, k", [(1, 1, 1), (5, 8, 8), (33, 32, 4), (17, 40, 3), (9, 64, 16), (257, 100, 6), (64, 128, 8),
                                                (31, 256, 8), (12, 333, 10), (20, 512, 16), (0, 16, 2), (1500, 32, 4)])
def test_scores_choice_and_gradient(dtype, score, renormalize, tokens, experts, k):
    logits = _logits(tokens, experts, dtype)
    _check(logits, k, score=score, renormalize=renormalize)
    bias = _logits(1, experts, torch.float32, 3, 0.1)[0]
    _check(logits, k, score=score, renormalize=renormalize, bias=bias, scale=2.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("experts, groups, kept, top, k", [(256, 8, 4, 2, 8), (64, 8, 3, 1, 6), (32, 4, 1, 2, 8), (160, 8, 3, 1, 6), (8, 8, 2, 2, 2),
                                                           (512, 32, 5, 2, 16), (96, 3, 3, 2, 5), (60, 4, 2, 2, 7)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups(dtype, with_bias, experts, groups, kept, top, k, score):
    logits = _logits(211, experts, dtype, 1)
    bias = _logits(1, experts, torch.float32, 4, 0.1)[0] if with_bias else None
    _check(logits, k, score=score, bias=bias, num_groups=groups, groups_kept=kept, group_top=top)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_equal_and_nearly_equal_keys(score):
    # a bias of zeros and logits of few values: equals go to the lowest index
    logits = torch.randint(-2, 3, (400, 48), generator=torch.Generator().manual_seed(0)).float().cuda()
    zero = torch.zeros(48, device="cuda")
    for bias in (None, zero):
        _check(logits, 7, score=score, bias=bias)
        _check(logits, 7, score=score, bias=bias, num_groups=6, groups_kept=3, group_top=2)
    # zeros of both signs are one number
    signed = torch.where(torch.rand(300, 48, generator=torch.Generator().manual_seed(5)) < 0.5, 0.0, -0.0)
    signed[:, 40:] = -1.0
    for l in (signed.cuda(), signed.cuda().bfloat16()):
        for bias in (None, zero):
            _check(l, 7, score=score, bias=bias)
            _check(l, 7, score=score, bias=bias, num_groups=6, groups_kept=3, group_top=1)
    # neighbours one step of fp32 apart, whose scores fp32 does not tell apart
    g = torch.Generator().manual_seed(1)
    base = torch.tensor([4.0, 1.0, -6.0, -30.0])[torch.randint(0, 4, (600, 1), generator=g)]
    steps = torch.stack([torch.randperm(64, generator=g) for _ in range(600)])
    near = (base.view(torch.int32) + steps.int()).view(torch.float32).cuda()
    _check(near, 8, score=score, bias=torch.zeros(64, device="cuda"))
    # a bias that brings different scores within a few steps of one another
    l = _logits(300, 64, torch.float32, 2)
    s = torch.sigmoid(l[0].double()) if score == "sigmoid" else torch.softmax(l[0].double(), -1)
    wobble = torch.randint(-4, 5, (64,), generator=g).double().cuda() * 2.0 ** -25
    _check(l, 8, score=score, bias=(0.75 - s + wobble).float())
    _check(l, 8, score=score, bias=(0.75 - s + wobble).float(), num_groups=8, groups_kept=4, group_top=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_choice_of_one_has_its_whole_weight_and_no_gradient(score, dtype):
    for experts, renormalize in ((40, True), (256, True), (1, True)) + (((1, False),) if score == "softmax" else ()):
        leaf = _logits(500, experts, dtype, std=4.0).requires_grad_(True)
        _, weights = routing.route_experts(leaf, 1, score=score, renormalize=renormalize, scale=2.5)
        assert (weights == 2.5).all()
        (dl,) = torch.autograd.grad(weights, leaf, _logits(500, 1, torch.float32, 6))
        assert (dl == 0).all()


@pytest.mark.parametrize("k", [1, 3])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_large_score_under_a_negative_bias(score, k):
    # the error of expert 7's key is that of a score near 1, far above its neighbours': it passes them in steps of 1e-9
    g = torch.Generator().manual_seed(3)
    rows, experts = 3000, 64
    l = torch.randn(rows, experts, generator=g) * 0.01 - 7.0
    l[:, 7] = (3.0 if score == "softmax" else 2.0) + torch.arange(rows) * 2.0 ** -22
    l = l.cuda()
    s = torch.softmax(l.double(), -1) if score == "softmax" else torch.sigmoid(l.double())
    bias = torch.zeros(experts, device="cuda")
    middle = s[:, [e for e in range(experts) if e != 7]].topk(k, -1).values[:, -1].mean()
    for shift in (-3e-4, -2e-5, 0.0, 2e-5):
        bias[7] = (middle - s[rows // 2, 7] + shift).float()
        _check(l, k, score=score, bias=bias)
        _check(l, k, score=score, bias=bias, num_groups=8, groups_kept=7, group_top=1)


def test_a_choice_that_ends_among_equals():
    # the last choice and its successor are the same number; behind them one a step above or below it
    g = torch.Generator().manual_seed(4)
    l = torch.randn(2000, 64, generator=g) - 3.0
    at = torch.stack([torch.randperm(64, generator=g)[:4] for _ in range(2000)])
    l.scatter_(1, at[:, :3], 1.0)
    step = torch.tensor([1.0 + 2.0 ** -23, 1.0 - 2.0 ** -24])[torch.randint(0, 2, (2000,), generator=g)]
    l.scatter_(1, at[:, 3:], step.unsqueeze(1))
    for k in (1, 2, 3):
        _check(l.cuda(), k)
        _check(l.cuda(), k, bias=torch.zeros(64, device="cuda"))
        _check(l.cuda(), k, score="sigmoid", bias=torch.full((64,), 0.25, device="cuda"))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_masked_experts_and_tokens(score, renormalize):
    logits = _logits(64, 32, torch.float32)
    logits[0] = -torch.inf                       # nothing left: zero weights, zero gradient
    logits[1, 2:] = -torch.inf                   # fewer than k left
    logits[2, 5] = torch.finfo(torch.float32).min
    logits[3] = torch.finfo(torch.float32).min   # a mask of the type's lowest value
    logits[4, ::2] = -torch.inf
    bias = _logits(1, 32, torch.float32, 3, 0.1)[0]
    for b in (None, bias):
        leaf = logits.clone().requires_grad_(True)
        ids, weights = routing.route_experts(leaf, 4, score=score, renormalize=renormalize, bias=b)
        (dl,) = torch.autograd.grad(weights, leaf, torch.randn_like(weights))
        assert torch.isfinite(weights).all() and torch.isfinite(dl).all()
        assert (weights[0] == 0).all() and (dl[0] == 0).all()
        assert (ids.sort(-1).values.diff(dim=-1) > 0).all() and ids.min() >= 0 and ids.max() < 32
        keep = [1, 2, 4] + list(range(5, 64))
        want = route64(logits[keep], 4, score=score, renormalize=renormalize, bias=b)
        assert torch.equal(ids[keep].cpu().long(), want[0])
        assert ((weights[keep].detach().cpu().double() - want[1]).abs() <= want[1] * W + 1e-37).all()


def test_nan_and_infinite_logits_choose_different_experts_and_stay_in_their_row():
    clean = _logits(16, 64, torch.float32)
    logits = clean.clone()
    logits[3, 10], logits[5, 7], logits[7] = torch.nan, torch.inf, torch.nan
    bias = torch.zeros(64, device="cuda")
    for options in (dict(), dict(bias=bias), dict(bias=bias, score="sigmoid", num_groups=8, groups_kept=2, group_top=2)):
        ids, weights = routing.route_experts(logits, 6, **options)
        assert ids.min() >= 0 and ids.max() < 64 and (ids.sort(-1).values.diff(dim=-1) > 0).all()
        # a softmax with one NaN is NaN for every expert, and equals go to the lowest index
        spread = "bias" in options and "score" not in options
        assert ids[3, 0] == (0 if spread else 10) and torch.isnan(weights[3]).any()
        same = [i for i in range(16) if i not in (3, 5, 7)]
        want = routing.route_experts(clean, 6, **options)
        assert torch.equal(ids[same], want[0][same]) and torch.equal(weights[same], want[1][same])


def test_small_scores_keep_their_ratio():
    # all logits far below zero: the scores leave fp32, the chosen ones' ratio does not
    logits = (_logits(40, 64, torch.float32) - 200.0)
    _, weights = routing.route_experts(logits, 4, score="sigmoid")
    ids, want, _ = route64(logits + 180.0, 4, score="sigmoid")      # e^x / (1 + e^x) is e^x at both
    l = logits.cpu().double().gather(-1, ids)
    want = torch.softmax(l, -1)
    assert ((weights.cpu().double() - want).abs() <= want * 2.0 ** -15).all()   # arguments of 200: 200 2^-24 more, twice


def test_strides_leading_dimensions_and_streams():
    wide = _logits(60, 70, torch.float32)
    want = routing.route_experts(wide[:, :64].contiguous(), 5)
    for view in (wide[:, :64], wide[:, :64].t().contiguous().t(), wide[:, :64].view(3, 20, 64) if wide[:, :64].is_contiguous() else wide[:, :64]):
        got = routing.route_experts(view, 5)
        assert torch.equal(got[0].view(60, 5), want[0]) and torch.equal(got[1].view(60, 5), want[1])
    three = wide[:, :64].contiguous().view(3, 20, 64).requires_grad_(True)
    ids, weights = routing.route_experts(three, 5)
    assert ids.shape == weights.shape == (3, 20, 5)
    weights.sum().backward()
    assert three.grad.shape == three.shape
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = routing.route_experts(wide[:, :64], 5)
        plan = routing.expert_plan(got[0], 64)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(plan.slot, routing.expert_plan(want[0], 64).slot)


@pytest.mark.parametrize("score, renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_gradient_against_differences(score, renormalize):
    logits = _logits(7, 24, torch.float32).requires_grad_(True)
    ids, weights = routing.route_experts(logits, 5, score=score, renormalize=renormalize, scale=1.5)
    up = _logits(7, 5, torch.float32, 8)
    (dl,) = torch.autograd.grad(weights, logits, up)
    l, chosen, step = logits.detach().double(), ids.long(), 1e-4

    def value(x):
        s = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x)
        c = s.gather(-1, chosen)
        return ((c / c.sum(-1, keepdim=True) if renormalize else c) * 1.5 * up.double()).sum()
    for seed in range(4):
        v = _logits(7, 24, torch.float32, 20 + seed).double()
        along = (value(l + step * v) - value(l - step * v)) / (2 * step)
        assert abs((dl.double() * v).sum() - along) <= 1e-5 * up.double().norm() * v.norm()   # step^2 of third derivatives, fp32


def plan_by_hand(ids, experts, align, rows):
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    k = ids.shape[-1]
    valid = (flat >= 0) & (flat < experts)
    counts = np.bincount(flat[valid], minlength=experts)
    runs = np.maximum(-(-counts // align), 1) * align
    ends = np.cumsum(runs)
    position, slot = np.full(rows, -1), np.full(flat.size, -1)
    nxt = (ends - runs).copy()
    for i, e in enumerate(flat):
        if valid[i]:
            if nxt[e] < rows:
                position[nxt[e]], slot[i] = i, nxt[e]
            nxt[e] += 1
    return np.where(position < 0, -1, position // k), position, slot, ends, counts


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens, k, experts, align", [(0, 2, 4, 128), (1, 1, 1, 128), (7, 3, 5, 128), (300, 4, 32, 128), (512, 4, 16, 1),
                                                       (513, 4, 16, 32), (3000, 2, 1, 128), (5000, 8, 256, 128), (2600, 10, 512, 8),
                                                       (4099, 7, 1024, 128), (40000, 4, 33, 128),
                                                       (200000, 3, 17, 128), (70000, 8, 700, 32), (4096, 1, 8, 128), (4097, 1, 8, 128)])
def test_plan(tokens, k, experts, align, dtype):
    g = torch.Generator().manual_seed(tokens)
    ids = (torch.randn(tokens, k, generator=g).abs() * experts / 3).long().clamp_max(experts - 1).to(dtype)
    plan = routing.expert_plan(ids.cuda(), experts, align)
    rows = (tokens * k + experts * align) // align * align
    assert plan.token.shape == (rows,)
    for got, want in zip(plan, plan_by_hand(ids, experts, align, rows)):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), want)


def test_plan_of_slots_without_an_expert_and_of_a_short_buffer():
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-3, 12, (1500, 4), generator=g)
    ids[5] = torch.tensor([-1, 2 ** 40, -2 ** 40, 11])
    for rows in (None, 0, 1, 1000, 6000, 9999):
        plan = routing.expert_plan(ids.cuda(), 9, 128, rows)
        for got, want in zip(plan, plan_by_hand(ids, 9, 128, plan.token.numel())):
            assert np.array_equal(got.cpu().numpy(), want)
        assert rows is None or plan.token.numel() == rows


def test_captured_plans_keep_their_own_work_space():
    g = torch.Generator().manual_seed(4)
    a, b = (torch.randint(0, 64, (9000, 4), generator=g).int().cuda() for _ in range(2))
    routing.expert_plan(a, 64)
    graphs, plans = [], []
    for ids in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plans.append(routing.expert_plan(ids, 64))
        graphs.append(graph)
    new = torch.randint(0, 64, (9000, 4), generator=g).int().cuda()
    a.copy_(new)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.synchronize()
    for ids, plan in ((new, plans[0]), (b, plans[1])):
        assert all(torch.equal(x, y) for x, y in zip(plan, routing.expert_plan(ids, 64)))


def test_refusals():
    l = _logits(4, 32, torch.float32)
    for bad in (dict(top_k=0), dict(top_k=17), dict(top_k=2, score="tanh"), dict(top_k=2, num_groups=5), dict(top_k=2, num_groups=4, groups_kept=5),
                dict(top_k=2, num_groups=4, group_top=3), dict(top_k=9, num_groups=4, groups_kept=1), dict(top_k=2, bias=l[0, :31])):
        with pytest.raises(ValueError):
            routing.route_experts(l, **bad)
    with pytest.raises(ValueError):
        routing.route_experts(_logits(2, 513, torch.float32), 2)
    with pytest.raises(TypeError):
        routing.route_experts(l.half(), 2)
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for bad in (dict(num_experts=0), dict(num_experts=1025), dict(num_experts=4, align=0), dict(num_experts=4, rows=-1)):
        with pytest.raises(ValueError):
            routing.expert_plan(ids, **bad)
    with pytest.raises(TypeError):
        routing.expert_plan(ids.float(), 4)
