"""The operators of a mixture-of-experts block around the low-precision products, as plain cases that can be timed and
compared: each in its plain form (elementary tensor operations) and, with ``own`` set, as this package's calls.

* ``norm``   - root-mean-square norm of a token's row, with the residual's addition in front, forward and backward, or with
  its result as MXFP8 codes and scales (the operand of the block-scaled product);
* ``route``  - scores of the experts, the choice of ``top_k`` (bias for balance, groups of experts) and the chosen experts'
  weights, with the gradient of the router's logits;
* ``plan``   - rows of the expert-major, padded token buffer that the grouped products read, from the chosen experts;
* ``swiglu`` - the gated activation between the two grouped products, whose input is kept for the backward pass in 8 bits.

Every case is a dict of plain values; activations are N(0, 1), weights N(1, 0.1), upstream gradients N(0, 1e-3).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
ALIGN = 128
# exponent of the largest value and kept mantissa bits of the two 8-bit formats
FORMATS = {"e4m3": (8, 3, torch.float8_e4m3fn, 448.0), "e5m2": (15, 2, torch.float8_e5m2, 57344.0)}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _norm(rows, cols, out="same", dtype="bfloat16", weight_dtype="bfloat16", residual=True, backward=False, pitch=0):
    """``out``: "same" (the type of x), or the 8-bit format of the result; ``pitch``: columns between the rows of x."""
    return {"op": "norm", "rows": rows, "cols": cols, "out": out, "dtype": dtype, "weight_dtype": weight_dtype,
            "residual": residual, "backward": backward, "pitch": pitch}


def _route(tokens, experts, top_k, score="softmax", bias=False, num_groups=1, groups_kept=1, group_top=1, renormalize=True,
           scale=1.0, dtype="bfloat16", backward=True):
    return {"op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "score": score, "bias": bias,
            "num_groups": num_groups, "groups_kept": groups_kept, "group_top": group_top, "renormalize": renormalize,
            "scale": scale, "dtype": dtype, "backward": backward}


def _plan(tokens, top_k, experts, skew=0.0):
    """``skew``: how unevenly the experts are liked (standard deviation of their offsets in the logits)."""
    return {"op": "plan", "tokens": tokens, "top_k": top_k, "experts": experts, "skew": skew}


def _swiglu(rows, hidden, fmt="e4m3", backward=True):
    return {"op": "swiglu", "rows": rows, "hidden": hidden, "format": fmt, "backward": backward}


def listed():
    cases = {
        # a decoding step of a few sequences: residual, norm and the 8-bit operand of the next linear
        "norm_decode_mxfp8": _norm(7, 4096, out="e4m3"),
        # Llama-3-8B's layer at the benchmark's 8192 tokens, a training step
        "norm_train_8192x4096": _norm(8192, 4096, backward=True),
        # four sequences of 8192 tokens, master weights of the norm in fp32
        "norm_train_32768x4096": _norm(32768, 4096, weight_dtype="float32", backward=True),
        # evaluation at GPT-OSS-20B's width, an odd number of tokens, rows of a wider buffer
        "norm_mxfp8_odd_2880": _norm(16381, 2880, out="e5m2", pitch=64),
        # a debugging run in fp32: odd width, no residual
        "norm_train_fp32_1023x1537": _norm(1023, 1537, dtype="float32", weight_dtype="float32", residual=False, backward=True),
        # GPT-OSS-20B's router: 32 experts, softmax over the chosen four, a training step
        "route_softmax_16384x32": _route(16384, 32, 4),
        # many fine experts in groups: sigmoid scores, bias for balance, fp32 logits
        "route_groups_65536x256": _route(65536, 256, 8, score="sigmoid", bias=True, num_groups=8, groups_kept=4, group_top=2,
                                         scale=2.5, dtype="float32"),
        # a decoding step's router, probabilities over all experts
        "route_decode_5x128": _route(5, 128, 8, renormalize=False, backward=False),
        # GPT-OSS-20B's token path: 65 536 routed rows over 32 experts
        "plan_16384x4_32": _plan(16384, 4, 32),
        # many fine experts, unevenly liked
        "plan_32749x8_256": _plan(32749, 8, 256, skew=1.0),
        # the same block's activation: 65 536 routed rows and every expert's padding
        "swiglu_train_69632x2880": _swiglu(69632, 2880),
        # a short batch of a small model
        "swiglu_train_384x1056_e5m2": _swiglu(384, 1056, "e5m2"),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _spread(rng, low, high, step=1):
    """A multiple of ``step`` in [low, high], even over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high // step * step, max(-(-low // step) * step, int(round(v / step)) * step))


_MOST_NORM = 32768 * 4096
_MOST_SCORES = 65536 * 256
_MOST_ROUTED = 32749 * 8
_MOST_HIDDEN = 69632 * 2880


def draw(rng):
    op = rng.choice(["norm", "norm", "route", "route", "plan", "swiglu"])
    if op == "norm":
        out = rng.choice(["same", "same", "e4m3", "e5m2"])
        step = 1 if out == "same" and rng.random() < 0.3 else 32
        cols = _spread(rng, 64, 16384, step)
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        rows = _spread(rng, 1, max(1, min(32768, _MOST_NORM // cols // (2 if dtype == "float32" else 1))))
        return _norm(rows, cols, out, dtype, rng.choice(["bfloat16", "float32"]) if dtype == "bfloat16" else "float32",
                     rng.random() < 0.7, out == "same" and rng.random() < 0.7, rng.choice([0, 0, 8, 64, 5]))
    if op == "route":
        score = rng.choice(["softmax", "sigmoid"])
        num_groups = rng.choice([1, 1, 4, 8])
        experts = num_groups * (_spread(rng, 8, 512) if num_groups == 1 else _spread(rng, 4, 512 // num_groups))
        kept = 1 if num_groups == 1 else rng.randint(1, num_groups)
        most = min(16, kept * (experts // num_groups))
        dtype = rng.choice(["bfloat16", "float32"])
        tokens = _spread(rng, 1, max(1, min(65536, _MOST_SCORES // experts)))
        return _route(tokens, experts, rng.randint(1, most), score, rng.random() < 0.5, num_groups, kept,
                      1 if num_groups == 1 else rng.choice([1, 2]), rng.random() < 0.7, rng.choice([1.0, 2.5]), dtype,
                      rng.random() < 0.7)
    if op == "plan":
        experts, top_k = _spread(rng, 4, 512), rng.randint(1, 10)
        top_k = min(top_k, experts)
        return _plan(_spread(rng, 1, min(65536, _MOST_ROUTED // top_k)), top_k, experts, rng.choice([0.0, 1.0, 3.0]))
    hidden = _spread(rng, 64, 14336, 32)
    return _swiglu(_spread(rng, 1, min(69632, _MOST_HIDDEN // hidden)), hidden, rng.choice(["e4m3", "e5m2"]), rng.random() < 0.8)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _normal(gen, shape, std, dtype=torch.bfloat16, mean=0.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * std + mean).to(dtype)


def plan_rows(case):
    """Rows of a buffer that holds every expert's run, however the tokens are routed."""
    return (case["tokens"] * case["top_k"] + case["experts"] * ALIGN) // ALIGN * ALIGN


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    op = case["op"]
    if op == "norm":
        dt, rows, cols = getattr(torch, case["dtype"]), case["rows"], case["cols"]
        state["x"] = _normal(gen, (rows, cols + case["pitch"]), 1.0, dt)[:, :cols]
        state["w"] = _normal(gen, (cols,), 0.1, getattr(torch, case["weight_dtype"]), 1.0)
        state["res"] = _normal(gen, (rows, cols), 2.0, dt) if case["residual"] else None
        if case["backward"]:
            state["dy"] = _normal(gen, (rows, cols), 1e-3, dt)
            state["dr"] = _normal(gen, (rows, cols), 1e-3, dt) if case["residual"] else None
            for name in ("x", "w", "res"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
    elif op == "route":
        state["logits"] = _normal(gen, (case["tokens"], case["experts"]), 1.0, getattr(torch, case["dtype"]))
        state["bias"] = _normal(gen, (case["experts"],), 0.05, torch.float32) if case["bias"] else None
        if case["backward"]:
            state["dw"] = _normal(gen, (case["tokens"], case["top_k"]), 1e-2, torch.float32)
            state["logits"].requires_grad_(True)
    elif op == "plan":
        liked = torch.randn(case["experts"], generator=gen, device=DEVICE) * case["skew"]
        logits = torch.randn(case["tokens"], case["experts"], generator=gen, device=DEVICE) + liked
        state["ids"] = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]].to(torch.int32).contiguous()
    else:
        state["h"] = _normal(gen, (case["rows"], 2 * case["hidden"]), 1.0)
        if case["backward"]:
            state["dy"] = _normal(gen, (case["rows"], case["hidden"]), 1e-3)
            state["h"].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------------------------
# one pass: plain forms
# ---------------------------------------------------------------------------------------------
def _mxfp8_values(t, fmt):
    """``t`` (bf16 or fp32) as the values of its 8-bit codes: one power-of-two scale for 32 neighbours, from the exponent of
    their largest magnitude, rounded to the format's mantissa first."""
    tmax, mbits, f8, most = FORMATS[fmt]
    blocks = t.unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True).float().view(torch.int32)
    kept = amax + (1 << (22 - mbits))
    scale = (((kept >> 23) - tmax).clamp_min(1) << 23).view(torch.float32)
    codes = (blocks.float() / scale).clamp(-most, most).to(f8)
    return (codes.float() * scale).flatten(-2)


def _plain_norm(state):
    case = state["case"]
    x, w, res = state["x"].detach(), state["w"].detach(), state["res"]
    # the stream after the addition is a tensor of x's type, and it is what the norm takes
    r = x if res is None else (x.float() + res.detach().float()).to(x.dtype)
    rf = r.float()
    rstd = torch.rsqrt((rf * rf).mean(-1, keepdim=True) + EPS)
    xhat = rf * rstd
    y = (xhat * w.float()).to(x.dtype)
    out = {"y": y if case["out"] == "same" else _mxfp8_values(y, case["out"]).to(torch.bfloat16)}
    if res is not None:
        out["r"] = r
    if case["backward"]:
        g = state["dy"].float()
        gw = g * w.float()
        dr = rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
        if res is not None:
            dr = dr + state["dr"].float()
        dr = dr.to(x.dtype)
        out["dx"], out["dw"] = dr, (g * xhat).sum(0).to(w.dtype)
        if res is not None:
            out["dres"] = dr
    return out


def _keys(l, case, bias):
    """What the experts are chosen by: the logits where that is the order of the scores, else scores and bias in 64 bits,
    because neighbours may be nearer than 32 bits tell apart."""
    if bias is None and case["group_top"] == 1:
        return l.double()
    l = l.double()
    s = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.exp(l - l.amax(-1, keepdim=True))
    if case["score"] == "softmax":
        s = s / s.sum(-1, keepdim=True)
    return s if bias is None else s + bias.double()


def _plain_route(state):
    case, logits, bias = state["case"], state["logits"].detach(), state["bias"]
    key = _keys(logits, case, bias)
    if case["num_groups"] > 1:
        groups = key.unflatten(-1, (case["num_groups"], -1))
        of_group = torch.sort(groups, dim=-1, descending=True).values[..., :case["group_top"]].sum(-1)
        kept = torch.sort(of_group, dim=-1, descending=True, stable=True).indices[:, :case["groups_kept"]]
        out_of = torch.ones_like(of_group, dtype=torch.bool).scatter_(1, kept, False)
        key = groups.masked_fill(out_of.unsqueeze(-1), -math.inf).flatten(-2)
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
    l = logits.float()
    if case["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        s = torch.exp(l - l.amax(-1, keepdim=True))
        s = s / s.sum(-1, keepdim=True)
    chosen = s.gather(1, ids)
    total = chosen.sum(-1, keepdim=True) if case["renormalize"] else 1.0
    out = {"ids": ids.to(torch.int32), "weights": chosen / total * case["scale"]}
    if case["backward"]:
        g = state["dw"] * case["scale"]
        if case["renormalize"]:
            g = (g - (g * (chosen / total)).sum(-1, keepdim=True)) / total
        ds = torch.zeros_like(s).scatter_(1, ids, g)
        dl = ds * s * (1.0 - s) if case["score"] == "sigmoid" else s * (ds - (ds * s).sum(-1, keepdim=True))
        out["dlogits"] = dl.to(logits.dtype)
    return out


def _plain_plan(state):
    case, ids = state["case"], state["ids"]
    experts, k, rows = case["experts"], case["top_k"], plan_rows(case)
    flat = ids.reshape(-1).long()
    counts = torch.zeros(experts, dtype=torch.int64, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    padded = ((counts + ALIGN - 1) // ALIGN * ALIGN).clamp_min(ALIGN)
    ends = torch.cumsum(padded, 0)
    order = torch.sort(flat, stable=True).indices
    sorted_ids = flat[order]
    place = (ends - padded)[sorted_ids] + torch.arange(flat.numel(), device=flat.device) - (torch.cumsum(counts, 0) - counts)[sorted_ids]
    position = torch.full((rows,), -1, dtype=torch.int64, device=flat.device)
    position[place] = order
    slot = torch.empty_like(flat)
    slot[order] = place
    token = torch.where(position < 0, position, position // k)
    return {"token": token.int(), "position": position.int(), "slot": slot.int(), "offs": ends.int(), "counts": counts.int()}


def _plain_swiglu(state):
    case, h = state["case"], state["h"].detach()
    n = case["hidden"]
    g, u = h[:, :n].float(), h[:, n:].float()
    # the package's activation rounds the gate's SiLU to bf16, as the product of two tensors does
    out = {"y": ((g / (1.0 + torch.exp(-g))).to(torch.bfloat16).float() * u).to(torch.bfloat16)}
    if case["backward"]:
        kept = _mxfp8_values(h, case["format"])
        g, u, d = kept[:, :n], kept[:, n:], state["dy"].float()
        s = 1.0 / (1.0 + torch.exp(-g))
        out["dh"] = torch.cat([d * u * s * (1.0 + g * (1.0 - s)), d * g * s], -1).to(torch.bfloat16)
    return out


# ---------------------------------------------------------------------------------------------
# one pass: this package's calls
# ---------------------------------------------------------------------------------------------
def _own_norm(state):
    from alto_b200 import mxfp8, norm
    case, x, w, res = state["case"], state["x"], state["w"], state["res"]
    if case["out"] != "same":
        got = norm.rms_norm_mxfp8(x, w, EPS, residual=res, mxfp_format=case["out"])
        out = {"y": mxfp8.convert_from_mxfp8(got[0], got[1], output_dtype=torch.bfloat16)}
        if res is not None:
            out["r"] = got[2]
        return out
    got = norm.rms_norm(x, w, EPS, residual=res)
    out = {"y": got} if res is None else {"y": got[0], "r": got[1]}
    if case["backward"]:
        if res is None:
            out["dx"], out["dw"] = torch.autograd.grad((out["y"],), (x, w), (state["dy"],))
        else:
            out["dx"], out["dw"], out["dres"] = torch.autograd.grad((out["y"], out["r"]), (x, w, res), (state["dy"], state["dr"]))
        out["y"] = out["y"].detach()
        if res is not None:
            out["r"] = out["r"].detach()
    return out


def _own_route(state):
    from alto_b200 import routing
    case = state["case"]
    ids, weights = routing.route_experts(state["logits"], case["top_k"], score=case["score"], bias=state["bias"],
                                         num_groups=case["num_groups"], groups_kept=case["groups_kept"],
                                         group_top=case["group_top"], renormalize=case["renormalize"], scale=case["scale"])
    out = {"ids": ids, "weights": weights}
    if case["backward"]:
        (out["dlogits"],) = torch.autograd.grad((weights,), (state["logits"],), (state["dw"],))
        out["weights"] = weights.detach()
    return out


def _own_plan(state):
    from alto_b200 import routing
    plan = routing.expert_plan(state["ids"], state["case"]["experts"])
    return {"token": plan.token, "position": plan.position, "slot": plan.slot, "offs": plan.offs, "counts": plan.counts}


def _own_swiglu(state):
    from alto_b200 import swiglu
    case, h = state["case"], state["h"]
    y = swiglu.swiglu(h, checkpoint=case["format"])
    if not case["backward"]:
        return {"y": y}
    (dh,) = torch.autograd.grad((y,), (h,), (state["dy"],))
    return {"y": y.detach(), "dh": dh}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "route": _own_route, "plan": _own_plan, "swiglu": _own_swiglu}[op](state)
    return {"norm": _plain_norm, "route": _plain_route, "plan": _plain_plan, "swiglu": _plain_swiglu}[op](state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["cols"]
        b = 2 if case["dtype"] == "bfloat16" else 4
        wb = (2 if case["weight_dtype"] == "bfloat16" else 4) * case["cols"]
        res = 1 if case["residual"] else 0
        # x (and the residual) in, the result (and the stream) out
        total = n * b * (1 + 2 * res) + wb + (n * b if case["out"] == "same" else n + n // 32 + 2 * n)
        flops = 6 * n
        if case["backward"]:
            # the normed rows and the upstream gradients in, one gradient of the rows out
            total += n * b * (3 + res) + 2 * wb
            flops += 12 * n
        return {"bytes": total, "flops": flops}
    if op == "route":
        n, tk = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        b = 2 if case["dtype"] == "bfloat16" else 4
        total = n * b + 8 * tk
        if case["backward"]:
            total += n * b + 8 * tk + (n * b if case["score"] == "softmax" and not case["renormalize"] else tk * b)
        return {"bytes": total, "flops": 8 * n}
    if op == "plan":
        tk = case["tokens"] * case["top_k"]
        return {"bytes": 8 * tk + 8 * plan_rows(case) + 8 * case["experts"], "flops": 8 * tk}
    n = case["rows"] * case["hidden"]
    if not case["backward"]:
        return {"bytes": 6 * n, "flops": 8 * n}
    kept = 2 * n + n // 16
    return {"bytes": 6 * n + 2 * kept + 6 * n, "flops": 30 * n}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_codes(t, fmt):
    """Values of the 8-bit codes of ``t``, by comparing with the format's grid."""
    tmax, mbits, _, most = FORMATS[fmt]
    blocks = t.double().reshape(*t.shape[:-1], t.shape[-1] // 32, 32)
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1, keepdim=True))          # in [1/2, 1), so 2^(exponent - 1)
    up = (mantissa * 2.0 + 2.0 ** -(mbits + 1) >= 2.0).to(exponent.dtype)
    scale = torch.exp2((exponent - 1 + up - tmax).clamp_min(-126).double())
    v = (blocks / scale).clamp(-most, most)
    _, e = torch.frexp(v)
    least = {"e4m3": -6, "e5m2": -14}[fmt]
    step = torch.exp2((e - 1).clamp_min(least).double() - mbits)
    return (torch.round(v / step) * step).clamp(-most, most).mul(scale).reshape(t.shape)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "route": _exact_route, "plan": _exact_plan, "swiglu": _exact_swiglu}[case["op"]](case, state)


def _exact_norm(case, state):
    x, w = state["x"], state["w"].double()
    stream = x if state["res"] is None else (x.double() + state["res"].double()).to(x.dtype)
    d = stream.double()
    root = torch.sqrt(d.pow(2).sum(1) / case["cols"] + EPS).unsqueeze(1)
    y = d / root * w
    out = {"y": y if case["out"] == "same" else _exact_codes(y.to(x.dtype), case["out"])}
    if state["res"] is not None:
        out["r"] = stream.double()
    if case["backward"]:
        up = state["dy"].double()
        direct = up * w / root
        along = (direct * d).sum(1, keepdim=True) / (case["cols"] * root * root)
        grad = direct - d * along
        if state["res"] is not None:
            grad = grad + state["dr"].double()
            out["dres"] = grad
        out["dx"], out["dw"] = grad, torch.einsum("rc,rc->c", up, d / root)
    return {name: out[name] for name in ("y", "r", "dx", "dw", "dres") if name in out}


def _exact_route(case, state):
    l = state["logits"].double()
    score = torch.softmax(l, 1) if case["score"] == "softmax" else 1.0 / (1.0 + torch.exp(-l))
    by_logits = state["bias"] is None and case["group_top"] == 1
    key = l.clone() if by_logits else (score if state["bias"] is None else score + state["bias"].double())
    size = case["experts"] // case["num_groups"]
    if case["num_groups"] > 1:
        best = torch.topk(key.reshape(-1, case["num_groups"], size), min(case["group_top"], size), dim=2).values.sum(2)
        order = torch.argsort(-best, dim=1, stable=True)
        left = torch.zeros_like(best).scatter(1, order[:, :case["groups_kept"]], 1.0)
        key = torch.where(left.repeat_interleave(size, 1) > 0, key, torch.full_like(key, -math.inf))
    ids = torch.argsort(-key, dim=1, stable=True)[:, :case["top_k"]]
    taken = torch.gather(score, 1, ids)
    weights = case["scale"] * (taken / taken.sum(1, keepdim=True) if case["renormalize"] else taken)
    out = {"ids": ids.to(torch.int32), "weights": weights}
    if case["backward"]:
        g = state["dw"].double()
        dl = torch.zeros_like(l)
        if case["score"] == "softmax":
            # dw_i / dl_e = w_i (1[i = e] - p_e), with p over the chosen alone where they are renormalised
            dot = (g * weights).sum(1, keepdim=True)
            if case["renormalize"]:
                dl.scatter_(1, ids, weights * g - weights / case["scale"] * dot)
            else:
                dl = -score * dot
                dl.scatter_add_(1, ids, weights * g)
        else:
            slope = 1.0 - taken
            if case["renormalize"]:
                dl.scatter_(1, ids, slope * weights * (g - (g * weights).sum(1, keepdim=True) / case["scale"]))
            else:
                dl.scatter_(1, ids, slope * weights * g)
        out["dlogits"] = dl
    return out


def _exact_plan(case, state):
    import numpy as np
    ids = state["ids"].cpu().numpy().reshape(-1)
    counts = np.bincount(ids, minlength=case["experts"])
    runs = np.maximum(-(-counts // ALIGN), 1) * ALIGN
    ends = np.cumsum(runs)
    position = np.full(plan_rows(case), -1, dtype=np.int32)
    slot = np.empty(ids.size, dtype=np.int32)
    for e in range(case["experts"]):
        of_expert = np.flatnonzero(ids == e)
        first = ends[e] - runs[e]
        position[first:first + of_expert.size] = of_expert
        slot[of_expert] = np.arange(first, first + of_expert.size)
    token = np.where(position < 0, -1, position // case["top_k"]).astype(np.int32)
    got = {"token": token, "position": position, "slot": slot, "offs": ends.astype(np.int32), "counts": counts.astype(np.int32)}
    return {name: torch.from_numpy(v).to(DEVICE) for name, v in got.items()}


def _exact_swiglu(case, state):
    n, h = case["hidden"], state["h"]
    gate, up = h[:, :n].double(), h[:, n:].double()
    out = {"y": (gate * torch.sigmoid(gate)).to(torch.bfloat16).double() * up}
    del gate, up
    if case["backward"]:
        d, kept = state["dy"].double(), torch.empty(h.shape, dtype=torch.float64, device=h.device)
        for first in range(0, h.shape[0], 8192):
            kept[first:first + 8192] = _exact_codes(h[first:first + 8192], case["format"])
        gate, up = kept[:, :n], kept[:, n:]
        s = torch.sigmoid(gate)
        dh = torch.empty_like(kept)
        dh[:, n:] = d * gate * s
        dh[:, :n] = d * up * (s + gate * s * (1.0 - s))
        out["dh"] = dh
    return out
