"""The operators of a step in 8-bit floating point with one fp32 scale for each block of 128, as plain cases that can be
timed and compared: each in its plain form (elementary tensor operations) and, with ``own`` set, as this package's calls.

* ``linear``  - y = x W^T with both operands in 8 bits: a training step with the gradients of x and W, or serving, where the
  weight is there as codes and scales;
* ``grouped`` - the same for the rows of several experts, as many rows an expert as there are (none, too); rows behind the
  last expert give zeros;
* ``clip``    - the norm of all gradients together and the gradients scaled to a largest norm.

A block of 128 numbers along the reduced dimension (128 x 128 of a weight) has the scale s = max(|largest|, 1e-12) / top, top
being the format's largest number, and the codes of x / s, both quotients in fp32.  Along tokens the blocks begin at an
expert's first row.  Activations are N(0, 1) with some features ten times as large, weights N(0, 0.02), upstream gradients
N(0, 1e-3).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 128
LEAST = 1e-12
FORMATS = {"e4m3": (torch.float8_e4m3fn, 448.0), "e5m2": (torch.float8_e5m2, 57344.0)}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _linear(tokens, k, n, train=True, fmt="e4m3", dtype="bfloat16"):
    return {"op": "linear", "tokens": tokens, "k": k, "n": n, "train": train, "format": fmt, "dtype": dtype}


def _grouped(rows, experts, k, n, train=True, fmt="e4m3", dtype="bfloat16", skew=0.5, spare=0):
    """``skew``: how unevenly the experts are liked (standard deviation of their offsets in the logits); ``spare``: rows of the
    buffer behind the last expert's."""
    return {"op": "grouped", "rows": rows, "experts": experts, "k": k, "n": n, "train": train, "format": fmt, "dtype": dtype,
            "skew": skew, "spare": spare}


def _clip(shapes, dtype="bfloat16", layers=1, tensors=0, elements=0, norm="2", clips=True):
    """``shapes``: "decoder" (the parameters of ``layers`` decoder layers of width 4096) or "many" (``tensors`` of them with
    ``elements`` numbers together, sizes spread over their logarithm); ``dtype``: one type, or "mixed" (bf16 and fp32)."""
    return {"op": "clip", "shapes": shapes, "dtype": dtype, "layers": layers, "tensors": tensors, "elements": elements,
            "norm": norm, "clips": clips}


def listed():
    cases = {
        # one sequence's next token through Llama-3-8B's up projection
        "linear_decode_1x4096x14336": _linear(1, 4096, 14336, train=False),
        # a batch of sequences that each add a token, the attention's output projection
        "linear_decode_24x4096x4096": _linear(24, 4096, 4096, train=False),
        # a prompt of an odd length
        "linear_prompt_1999x4096x14336": _linear(1999, 4096, 14336, train=False),
        # the benchmark's linear, a training step
        "linear_train_8192x4096x14336": _linear(8192, 4096, 14336),
        # GPT-OSS-20B's widths (the last block has 64 numbers), a short and odd batch, gradients' format
        "linear_train_1021x2880x5760_e5m2": _linear(1021, 2880, 5760, fmt="e5m2"),
        # a debugging run in fp32
        "linear_train_fp32_513x1040x768": _linear(513, 1040, 768, dtype="float32"),
        # GPT-OSS-20B's experts at a decoding step: 16 tokens to 4 experts each
        "grouped_decode_64_32x2880x5760": _grouped(64, 32, 2880, 5760, train=False),
        # the same block's training step: 65 536 routed rows over 32 experts
        "grouped_train_65536_32x2880x5760": _grouped(65536, 32, 2880, 5760),
        # many small experts, unevenly liked, some without a row; a buffer with room to spare
        "grouped_train_3001_64x512x1024": _grouped(3001, 64, 512, 1024, skew=1.5, spare=100),
        # gradients of four decoder layers in bf16
        "clip_decoder_4": _clip("decoder", layers=4),
        # a model's small parameters, fp32 and bf16, not above the largest norm
        "clip_many_2000_mixed": _clip("many", "mixed", tensors=2000, elements=40_000_000, clips=False),
        # adapters of a small model
        "clip_many_60": _clip("many", "float32", tensors=60, elements=200_000),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _spread(rng, low, high, step=1):
    """A multiple of ``step`` in [low, high], even over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high // step * step, max(-(-low // step) * step, int(round(v / step)) * step))


_MOST_LINEAR = 8192 * 4096 * 14336
_MOST_GROUPED = 65536 * 2880 * 5760
_MOST_EXPERTS = 32 * 2880 * 5760
_MOST_CLIP = 800_000_000


def draw(rng):
    op = rng.choice(["linear", "linear", "grouped", "grouped", "clip"])
    fmt = rng.choice(["e4m3", "e4m3", "e5m2"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if op == "linear":
        k, n = _spread(rng, 64, 16384, 16), _spread(rng, 64, 16384, 16)
        train = rng.random() < 0.5
        most = max(1, min(32768, _MOST_LINEAR // (k * n) // (2 if dtype == "float32" else 1)))
        return _linear(_spread(rng, 1, most), k, n, train, fmt, dtype)
    if op == "grouped":
        experts = _spread(rng, 2, 128)
        k, n = _spread(rng, 64, 6144, 16), _spread(rng, 64, 6144, 16)
        experts = max(1, min(experts, _MOST_EXPERTS // (k * n)))
        train = rng.random() < 0.5
        most = max(1, min(65536, _MOST_GROUPED // (k * n) // (2 if dtype == "float32" else 1)))
        return _grouped(_spread(rng, 1, most), experts, k, n, train, fmt, dtype, rng.choice([0.0, 0.5, 1.5]), rng.choice([0, 0, 77]))
    norm = rng.choice(["2", "2", "2", "inf"])
    dtype = rng.choice(["bfloat16", "float32", "mixed"])
    if rng.random() < 0.3:
        return _clip("decoder", dtype, layers=rng.choice([1, 1, 2] if dtype != "bfloat16" else [1, 2, 3]), norm=norm, clips=rng.random() < 0.6)
    tensors = _spread(rng, 1, 4000)
    return _clip("many", dtype, tensors=tensors, elements=_spread(rng, 16 * tensors, _MOST_CLIP // 4), norm=norm, clips=rng.random() < 0.6)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _normal(gen, shape, std, dtype):
    return (torch.randn(shape, generator=gen, device=DEVICE) * std).to(dtype)


def _activations(gen, rows, k, dtype):
    loud = torch.where(torch.rand(k, generator=gen, device=DEVICE) < 0.01, 10.0, 1.0)
    return (torch.randn(rows, k, generator=gen, device=DEVICE) * loud).to(dtype)


def expert_counts(case, seed):
    """Rows of each expert, their sum the case's rows: every row's expert is drawn by the experts' softmax."""
    rng = random.Random(seed)
    liked = [math.exp(rng.gauss(0.0, case["skew"])) for _ in range(case["experts"])]
    counts = [0] * case["experts"]
    for e in rng.choices(range(case["experts"]), liked, k=case["rows"]):
        counts[e] += 1
    return counts


def clip_sizes(case):
    if case["shapes"] == "decoder":
        layer = [4096 * 4096, 1024 * 4096, 1024 * 4096, 4096 * 4096, 14336 * 4096, 14336 * 4096, 4096 * 14336, 4096, 4096]
        return layer * case["layers"]
    rng = random.Random(case["tensors"])
    shares = [math.exp(rng.uniform(0.0, 8.0)) for _ in range(case["tensors"])]
    total = sum(shares)
    return [max(1, int(s / total * case["elements"])) for s in shares]


def _split(flat, sizes):
    return list(torch.split(flat, sizes))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    if case["op"] == "clip":
        sizes = clip_sizes(case)
        kinds = {"mixed": [torch.bfloat16, torch.float32]}.get(case["dtype"]) or [getattr(torch, case["dtype"])]
        # gradients lie one behind the other in a buffer of their type; the clipped ones have such buffers too
        by_kind = [sizes[i::len(kinds)] for i in range(len(kinds))]
        state["flat"] = [_normal(gen, (sum(s),), 1e-3, t) for s, t in zip(by_kind, kinds)]
        state["out_flat"] = [torch.empty_like(f) for f in state["flat"]]
        state["grads"] = [g for f, s in zip(state["flat"], by_kind) for g in _split(f, s)]
        state["outs"] = [g for f, s in zip(state["out_flat"], by_kind) for g in _split(f, s)]
        largest = 4.5e-3 if case["norm"] == "inf" else 1e-3 * math.sqrt(sum(sizes))
        state["max_norm"] = largest * (0.3 if case["clips"] else 4.0)
        return state
    dt, k, n = getattr(torch, case["dtype"]), case["k"], case["n"]
    if case["op"] == "linear":
        rows, shape = case["tokens"], (n, k)
    else:
        counts = expert_counts(case, seed)
        rows, shape = case["rows"] + case["spare"], (case["experts"], n, k)
        state["offs"] = torch.tensor(counts, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEVICE)
        state["most"] = max(counts)
    state["x"] = _activations(gen, rows, k, dt)
    w = _normal(gen, shape, 0.02, dt)
    if case["train"]:
        # an expert's weight lies as the grouped product takes it, [k, n]
        state["w"] = w if case["op"] == "linear" else w.transpose(1, 2).contiguous()
        state["dy"] = _normal(gen, (rows, n), 1e-3, dt)
        state["x"].requires_grad_(True)
        state["w"].requires_grad_(True)
    else:
        state["w_codes"], state["w_scales"] = _codes(w, case["format"], square=True)
    return state


# ---------------------------------------------------------------------------------------------
# one pass: plain forms
# ---------------------------------------------------------------------------------------------
def _blocks(t, square):
    """t in whole blocks of 128 (zeros behind its end): [..., blocks, 128], or [..., blocks, 128, blocks, 128]."""
    r, c = -t.shape[-2] % BLOCK, -t.shape[-1] % BLOCK
    t = torch.nn.functional.pad(t, (0, c, 0, r if square else 0))
    t = t.unflatten(-1, (-1, BLOCK))
    return t.unflatten(-3, (-1, BLOCK)) if square else t


def _unblocked(b, rows, cols, square):
    return (b.flatten(-2).flatten(-3, -2) if square else b.flatten(-2))[..., :rows, :cols]


def _codes(t, fmt, square=False):
    """(codes, scales) of t along its last dimension, or of its squares of 128 x 128."""
    f8, top = FORMATS[fmt]
    b = _blocks(t.float(), square)
    dims = (-3, -1) if square else (-1,)
    s = b.abs().amax(dims, keepdim=True).clamp_min(LEAST) / torch.full((), top, device=t.device)
    codes = _unblocked((b / s).clamp(-top, top), t.shape[-2], t.shape[-1], square).to(f8)
    return codes.contiguous(), (s.squeeze(-1).squeeze(-2) if square else s.squeeze(-1)).contiguous()


def _values(codes, scales, square=False):
    """What codes and scales stand for, in fp32."""
    b = _blocks(codes.float(), square)
    s = scales.unsqueeze(-1)
    return _unblocked(b * (s.unsqueeze(-3) if square else s), codes.shape[-2], codes.shape[-1], square)


def _through_codes(t, fmt, square=False):
    return _values(*_codes(t, fmt, square), square)


def _plain_linear(state):
    case, x = state["case"], state["x"].detach()
    fmt = case["format"]
    w = _through_codes(state["w"].detach(), fmt, True) if case["train"] else _values(state["w_codes"], state["w_scales"], True)
    out = {"y": (_through_codes(x, fmt) @ w.t()).to(x.dtype)}
    if case["train"]:
        dy = state["dy"]
        out["dx"] = (_through_codes(dy, fmt) @ w).to(x.dtype)
        # blocks of 128 tokens
        out["dw"] = (_through_codes(dy.t(), fmt) @ _through_codes(x.t(), fmt).t()).to(x.dtype)
    return out


def _plain_grouped(state):
    case, x, offs = state["case"], state["x"].detach(), state["offs"].long()
    fmt, experts = case["format"], case["experts"]
    # [experts, most rows an expert has]: row of the buffer
    starts = torch.nn.functional.pad(offs, (1, 0))[:-1]
    place = starts[:, None] + torch.arange(max(state["most"], 1), device=x.device)
    there = place < offs[:, None]
    place = place.clamp_max(x.shape[0] - 1)

    def apart(t):
        return torch.where(there[..., None], t[place], torch.zeros((), dtype=t.dtype, device=t.device))

    # rows behind the last expert belong to none
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(offs, row, right=True)
    none = (expert >= experts)[:, None]
    expert = expert.clamp_max(experts - 1)
    at = (row - starts[expert]).clamp(0, place.shape[1] - 1)

    def together(t):
        return torch.where(none, torch.zeros((), dtype=t.dtype, device=t.device), t[expert, at])

    w = _through_codes(state["w"].detach(), fmt, True) if case["train"] else _values(state["w_codes"], state["w_scales"], True).transpose(1, 2)
    xs = apart(x)
    out = {"y": together(torch.bmm(_through_codes(xs, fmt), w)).to(x.dtype)}
    if case["train"]:
        dys = apart(state["dy"])
        out["dx"] = together(torch.bmm(_through_codes(dys, fmt), w.transpose(1, 2))).to(x.dtype)
        xt, dyt = _through_codes(xs.transpose(1, 2), fmt), _through_codes(dys.transpose(1, 2), fmt)
        out["dw"] = torch.bmm(xt, dyt.transpose(1, 2)).to(x.dtype)
    return out


def _plain_clip(state):
    case, grads = state["case"], state["grads"]
    if case["norm"] == "inf":
        norm = torch.stack([g.abs().amax().double() for g in grads]).amax()
    else:
        norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    factor = (state["max_norm"] / (norm + 1e-6)).clamp_max(1.0).float()
    return {"norm": norm.float(), "grads": [torch.cat([(g.float() * factor).to(g.dtype) for g in grads if g.dtype == f.dtype])
                                            for f in state["flat"]]}


# ---------------------------------------------------------------------------------------------
# one pass: this package's calls
# ---------------------------------------------------------------------------------------------
def _gradients(state, y):
    dx, dw = torch.autograd.grad((y,), (state["x"], state["w"]), (state["dy"],))
    return {"y": y.detach(), "dx": dx, "dw": dw}


def _own_linear(state):
    from alto_b200 import fp8_block
    if not state["case"]["train"]:
        return {"y": fp8_block.fp8_block_linear(state["x"], state["w_codes"], state["w_scales"])}
    return _gradients(state, fp8_block._to_fp8_block_then_scaled_mm(state["x"], state["w"], fp8_variant=state["case"]["format"]))


def _own_grouped(state):
    from alto_b200 import fp8_block, grouped
    if not state["case"]["train"]:
        return {"y": fp8_block.fp8_block_grouped_linear(state["x"], state["w_codes"], state["w_scales"], state["offs"])}
    return _gradients(state, grouped._quantize_then_fp8_block_scaled_grouped_mm(state["x"], state["w"], offs=state["offs"],
                                                                                fp8_variant=state["case"]["format"]))


def _own_clip(state):
    from alto_b200 import grad_clip
    norm = grad_clip.clip_grads(state["grads"], state["max_norm"], norm_type=float(state["case"]["norm"]), out=state["outs"])
    return {"norm": norm, "grads": state["out_flat"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "grouped": _own_grouped, "clip": _own_clip}[op](state)
    return {"linear": _plain_linear, "grouped": _plain_grouped, "clip": _plain_clip}[op](state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "clip":
        sizes = clip_sizes(case)
        b = {"bfloat16": 2, "float32": 4, "mixed": 3}[case["dtype"]]
        return {"bytes": 2 * b * sum(sizes), "flops": 3 * sum(sizes)}
    b = 2 if case["dtype"] == "bfloat16" else 4
    k, n = case["k"], case["n"]
    if case["op"] == "linear":
        rows, used, weight = case["tokens"], case["tokens"], k * n
    else:
        rows, used = case["rows"] + case["spare"], case["rows"]
        # an expert without rows is not read
        weight = k * n * sum(c > 0 for c in expert_counts(case, 0))
    if not case["train"]:
        return {"bytes": used * k * b + weight + rows * n * b, "flops": 2 * k * n * used}
    whole = k * n * (case["experts"] if case["op"] == "grouped" else 1)
    return {"bytes": used * k * b + weight * b + rows * n * b + used * n * b + rows * k * b + whole * b, "flops": 6 * k * n * used}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_values(t, fmt, dim):
    """Values of the codes of a matrix whose blocks lie along ``dim`` (None: squares); scale and quotient are fp32 numbers by
    definition, and a quotient of fp32 numbers in 64 bits, rounded to fp32, is the rounded quotient."""
    f8, top = FORMATS[fmt]
    d = t.double()
    rows, cols = d.shape
    br, bc = (BLOCK if dim != 1 else 1), (BLOCK if dim != 0 else 1)
    full = d.new_zeros(-(-rows // br) * br, -(-cols // bc) * bc)
    full[:rows, :cols] = d
    tiles = full.reshape(full.shape[0] // br, br, full.shape[1] // bc, bc)
    largest = torch.maximum(tiles.abs().amax(3).amax(1), torch.tensor(LEAST, dtype=torch.float32).double().to(d.device))
    s = (largest / top).float().double()[:, None, :, None]
    q = (tiles / s).float().clamp(-top, top).to(f8).double() * s
    return q.reshape(full.shape)[:rows, :cols]


def _exact_products(x, w, dy, fmt, w_values=None):
    wv = _exact_values(w, fmt, None) if w_values is None else w_values
    y = _exact_values(x, fmt, 1) @ wv.T
    if dy is None:
        return y, None, None
    return y, _exact_values(dy, fmt, 1) @ wv, _exact_values(dy, fmt, 0).T @ _exact_values(x, fmt, 0)


def _spread_scales(codes, scales):
    s = scales.double().repeat_interleave(BLOCK, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.double() * s


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"linear": _exact_linear, "grouped": _exact_grouped, "clip": _exact_clip}[case["op"]](case, state)


def _exact_linear(case, state):
    if not case["train"]:
        return {"y": _exact_products(state["x"], None, None, case["format"], _spread_scales(state["w_codes"], state["w_scales"]))[0]}
    y, dx, dw = _exact_products(state["x"], state["w"], state["dy"], case["format"])
    return {"y": y, "dx": dx, "dw": dw}


def _exact_grouped(case, state):
    x, ends = state["x"], [0] + state["offs"].tolist()
    y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=x.device)
    out = {"y": y}
    if case["train"]:
        out["dx"] = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        out["dw"] = torch.zeros(state["w"].shape, dtype=torch.float64, device=x.device)
    for e in range(case["experts"]):
        rows = slice(ends[e], ends[e + 1])
        if rows.start == rows.stop:
            continue
        if case["train"]:
            y[rows], out["dx"][rows], dw = _exact_products(x[rows], state["w"][e].T, state["dy"][rows], case["format"])
            out["dw"][e] = dw.T
        else:
            values = _spread_scales(state["w_codes"][e], state["w_scales"][e])
            y[rows] = _exact_products(x[rows], None, None, case["format"], values)[0]
    return out


def _exact_clip(case, state):
    if case["norm"] == "inf":
        norm = max(float(f.abs().max()) for f in state["flat"])
    else:
        norm = math.sqrt(math.fsum(float(f[i:i + (1 << 26)].double().pow(2).sum()) for f in state["flat"] for i in range(0, f.numel(), 1 << 26)))
    factor = min(1.0, state["max_norm"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [f.double() * factor for f in state["flat"]]}
