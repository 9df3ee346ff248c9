"""Performance cases of the 8-bit operators beside the EXL3 projections: what a program has the package do for the layers of a
checkpoint that stay in 8-bit floating point (e4m3 with one scale for each block of 128), and for the routing ahead of any
routed layer. A case is a dict of plain values. The kinds:

  route     `route`: a router's logits to expert numbers and scores.
  quantize  `quantize_fp8`: activations to e4m3 with one f32 scale for each 128 values of a row.
  linear    `linear_fp8`: y = x W^T, W e4m3 [out, in] with one f32 scale for each 128 x 128 block. `given`: x comes quantised.
  moe       `moe_fp8`: a routed SwiGLU layer for a few tokens, its experts in the same format. The router numbers
            experts * share experts; this device holds the first `experts` of them, as a rank of an expert-parallel layer does,
            and a slot whose expert is elsewhere adds nothing.

The definitions: a group's scale is the smallest power of two (from 2^-126 up) that brings its largest magnitude to 448 or less, its
values are e4m3(x / scale), to nearest even; a linear is the product of the values times their scales, rounded once; between
an expert's projections silu(gate) * up is quantised in the same way. A router picks the largest logits (with `bias` or `groups`: the largest score + bias, of the groups with the
largest sums of two), the lowest number where they tie, and scores them by softmax or sigmoid.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
GROUP = 128


def route(name, rows, experts, topk, dtype="f32", scoring="softmax", bias=False, groups=1, group_topk=1, renormalise=True, scale=1.0):
    return {"name": name, "kind": "route", "rows": rows, "experts": experts, "topk": topk, "dtype": dtype, "scoring": scoring, "bias": bias,
            "groups": groups, "group_topk": group_topk, "renormalise": renormalise, "scale": scale}


def quantize(name, rows, width, dtype="bf16"):
    return {"name": name, "kind": "quantize", "rows": rows, "in": width, "dtype": dtype}


def linear(name, rows, width, out, dtype="bf16", given=False):
    return {"name": name, "kind": "linear", "rows": rows, "in": width, "out": out, "dtype": dtype, "given": given}


def moe(name, rows, hidden, inter, experts, topk, dtype="bf16", share=1):
    return {"name": name, "kind": "moe", "rows": rows, "hidden": hidden, "inter": inter, "experts": experts, "topk": topk, "dtype": dtype,
            "share": share}


def listed():
    return [
        # the router of a 512-expert layer for one token of a decode step: all launch and latency
        route("route_1row", 1, 512, 10),
        # a long prompt through the grouped sigmoid router of a 256-expert layer
        route("route_groups_8192rows", 8192, 256, 8, "f32", "sigmoid", True, 8, 4, True, 2.5),
        # a decode batch of ragged size, experts no multiple of a warp, 16-bit logits
        route("route_ragged_777rows", 777, 160, 6, "bf16", "softmax", False, 1, 1, False),
        # one token's hidden state, quantised once for several projections
        quantize("quantize_1row", 1, 7168),
        # a long prompt's
        quantize("quantize_8192rows", 8192, 7168),
        # one attention projection of a 2048-wide model for one token: latency
        linear("linear_1row", 1, 2048, 2048),
        # the largest attention projection of a 7168-wide model for a decode batch of ragged size: the weight's bytes
        linear("linear_o_29rows", 29, 16384, 7168, "f16"),
        # a short prompt through a narrow projection whose width is no multiple of 128
        linear("linear_kv_200rows", 200, 7168, 576),
        # a long prompt through an up projection, its rows quantised for the gate projection too
        linear("linear_8192rows", 8192, 2048, 6144, "bf16", True),
        # a 512-expert top-10 layer for one token, and for a decode batch of ragged size
        moe("moe_1row", 1, 2048, 512, 512, 10),
        moe("moe_29rows", 29, 2048, 512, 512, 10, "f16"),
        # one rank's quarter of a 256-expert top-8 layer for a small decode batch
        moe("moe_shard_8rows", 8, 7168, 2048, 64, 8, "bf16", 4),
    ]


LINEAR_MOST = 8192 * 2048 * 6144
WEIGHT_MOST = 16384 * 7168
BANK_MOST = 64 * 3 * 7168 * 2048


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    return max(lo, GROUP * round(_log_int(rng, lo, hi) / GROUP))


def draw(rng):
    """One more case: rows log-uniform from one token to a prompt's (decode batches of 1..32 for the routed layer), widths in
    steps of 128 where a group's scale needs it, any number of outputs and experts, every type."""
    kind = rng.choice(("route", "quantize", "linear", "linear", "moe", "moe"))
    if kind == "route":
        rows = _log_int(rng, 1, 8192)
        topk = rng.randint(1, 16)
        dtype = rng.choice(("f32", "f32", "bf16", "f16"))
        scoring, renormalise = rng.choice(("softmax", "sigmoid")), rng.random() < 0.7
        scale = rng.choice((1.0, 2.5))
        if rng.random() < 0.4:
            groups = rng.choice((2, 4, 8))
            experts = groups * rng.randint(8, 64)
            group_topk = rng.randint((topk * groups + experts - 1) // experts, groups)
            return route("", rows, experts, topk, "f32", scoring, True, groups, group_topk, renormalise, scale)
        return route("", rows, _log_int(rng, max(8, topk), 512), topk, dtype, scoring, dtype == "f32" and rng.random() < 0.5, 1, 1, renormalise, scale)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "quantize":
        width = _width(rng, 128, 16384)
        return quantize("", min(_log_int(rng, 1, 8192), 8192 * 7168 // width), width, dtype)
    if kind == "linear":
        width = _width(rng, 128, 16384)
        out = min(_log_int(rng, 16, 24576), WEIGHT_MOST // width)
        if rng.random() < 0.5:
            out = max(GROUP, out // GROUP * GROUP)
        rows = _log_int(rng, 1, 32) if rng.random() < 0.5 else _log_int(rng, 33, 8192)
        return linear("", min(rows, LINEAR_MOST // (width * out)), width, out, dtype, rng.random() < 0.3 and dtype != "f32")
    hidden, inter = _width(rng, 256, 7168), _width(rng, 128, 2048)
    experts = min(_log_int(rng, 4, 512), BANK_MOST // (3 * hidden * inter))
    rows, topk = _log_int(rng, 1, 32), rng.randint(1, min(10, experts))
    share = rng.choice((1, 1, 2, 4)) if rows * topk >= 32 else 1  # enough slots that some are this device's
    return moe("", rows, hidden, inter, experts, topk, "bf16" if dtype == "f32" else dtype, share)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _weight(gen, shape, width):
    """What a block-quantised weight holds: values near normal that fill e4m3's range, and a scale for each 128 x 128 block
    that brings them to about 1 / sqrt(width)."""
    w = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(112.0).clamp_(-448.0, 448.0).to(E4M3)
    blocks = shape[:-2] + (-(-shape[-2] // GROUP), shape[-1] // GROUP)
    return w, (0.5 + torch.rand(blocks, generator=gen, device="cuda")) / (112.0 * math.sqrt(width))


def _activations(gen, rows, width, dtype):
    """Hidden states: normal, with a few channels much larger than the others, as they are in trained models."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    x *= torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    return x.to(DTYPES[dtype])


def _values(x):
    """(e4m3 values, f32 scales) of x's groups of 128 along its last axis."""
    g = x.float().unflatten(-1, (-1, GROUP))
    part, power = torch.frexp(g.abs().amax(-1).clamp_min(2.0 ** -126))  # 448 is 0.875 * 2^9
    scale = torch.ldexp(torch.ones_like(part), (power - 9 + (part > 0.875)).clamp_min(-126))
    return (g / scale[..., None]).to(E4M3).flatten(-2), scale


def prepare(case, seed):
    gen = _generator(seed)
    kind = case["kind"]
    if kind == "route":
        logits = torch.randn(case["rows"], case["experts"], generator=gen, device="cuda").to(DTYPES[case["dtype"]])
        bias = 0.1 * torch.randn(case["experts"], generator=gen, device="cuda") if case["bias"] else None
        return {"case": case, "logits": logits, "bias": bias}
    if kind == "quantize":
        return {"case": case, "x": _activations(gen, case["rows"], case["in"], case["dtype"])}
    if kind == "linear":
        x = _activations(gen, case["rows"], case["in"], case["dtype"])
        w, w_scale = _weight(gen, (case["out"], case["in"]), case["in"])
        state = {"case": case, "x": x, "w": w, "w_scale": w_scale}
        if case["given"]:
            state["q"], state["x_scale"] = _values(x)
        return state
    hidden, inter, experts, rows, topk = case["hidden"], case["inter"], case["experts"], case["rows"], case["topk"]
    proj = [SimpleNamespace(w=w, scale=s) for w, s in (_weight(gen, (experts, o, i), i) for o, i in ((inter, hidden), (inter, hidden), (hidden, inter)))]
    x = _activations(gen, rows, hidden, case["dtype"])
    logits = torch.randn(rows, experts * case["share"], generator=gen, device="cuda")
    scores, inds = torch.topk(torch.softmax(logits, -1), topk)
    return {"case": case, "x": x[None], "bank": SimpleNamespace(gate=proj[0], up=proj[1], down=proj[2]), "inds": inds.to(torch.int32)[None],
            "scores": (scores / scores.sum(-1, keepdim=True))[None]}


def _plain_route(state):
    c, x = state["case"], state["logits"].float()
    # 64 bits where a choice hangs on a sum: a score plus its bias next to another's
    s64 = torch.softmax(x.double(), -1) if c["scoring"] == "softmax" else torch.sigmoid(x.double())
    pick = x
    if c["bias"] or c["groups"] > 1:
        pick = s64 if state["bias"] is None else s64 + state["bias"].double()
        grouped = pick.unflatten(-1, (c["groups"], -1))
        best = grouped.sort(dim=-1, descending=True).values[..., :2].sum(-1).sort(dim=-1, descending=True, stable=True).indices[..., : c["group_topk"]]
        out = torch.ones(best.shape[0], c["groups"], dtype=torch.bool, device="cuda").scatter_(-1, best, False)
        pick = grouped.masked_fill(out[..., None], -math.inf).flatten(-2)
    inds = pick.sort(dim=-1, descending=True, stable=True).indices[..., : c["topk"]]
    scores = (torch.softmax(x, -1) if c["scoring"] == "softmax" else torch.sigmoid(x)).gather(-1, inds)
    if c["renormalise"]:
        scores = scores / scores.sum(-1, keepdim=True)
    return inds.to(torch.int32), scores * c["scale"]


def _dequantized(q, scale):
    return (q.float().unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)


def _dequantized_weight(w, scale):
    """[..., out, in] of e4m3 with one scale a 128 x 128 block, the last block of rows possibly short."""
    rows = scale.repeat_interleave(GROUP, -2)[..., : w.shape[-2], :]
    return _dequantized(w, rows)


def _plain_linear(state):
    q, s = (state["q"], state["x_scale"]) if state["case"]["given"] else _values(state["x"])
    y = torch.matmul(_dequantized(q, s), _dequantized_weight(state["w"], state["w_scale"]).T)
    return y.to(state["x"].dtype)


def _plain_moe(state):
    bank, inds = state["bank"], state["inds"][0]
    here = inds < bank.gate.w.shape[0]
    used, at = torch.unique(torch.where(here, inds, 0), return_inverse=True)

    def weight(p):
        return _dequantized_weight(p.w.view(torch.uint8)[used].view(E4M3), p.scale[used]).transpose(-1, -2)

    x = _dequantized(*_values(state["x"][0]))
    gate, up = torch.matmul(x, weight(bank.gate)), torch.matmul(x, weight(bank.up))
    h = _dequantized(*_values(gate * torch.sigmoid(gate) * up))
    down = torch.matmul(h, weight(bank.down))  # [used, rows, hidden]
    slots = down[at, torch.arange(inds.shape[0], device="cuda")[:, None]]
    y = (torch.where(here, state["scores"][0], 0.0)[..., None] * slots).sum(1)
    return y.to(state["x"].dtype)[None]


def run(state):
    kind = state["case"]["kind"]
    if own:
        import turboexl3_b200 as t3
        c = state["case"]
        if kind == "route":
            return t3.route(state["logits"], c["topk"], c["scoring"], state["bias"], c["groups"], c["group_topk"], c["renormalise"], c["scale"])
        if kind == "quantize":
            return t3.quantize_fp8(state["x"])
        if kind == "moe":
            return t3.moe_fp8(state["x"], state["bank"], state["inds"], state["scores"])
        if c["given"]:
            return t3.linear_fp8(state["q"], state["w"], state["w_scale"], state["x_scale"], state["x"].dtype)
        return t3.linear_fp8(state["x"], state["w"], state["w_scale"])
    if kind == "route":
        return _plain_route(state)
    if kind == "quantize":
        return _values(state["x"])
    return _plain_linear(state) if kind == "linear" else _plain_moe(state)


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "f32" else 2
    rows = case["rows"]
    if kind == "route":
        e = case["experts"]
        return {"bytes": rows * (e * size + case["topk"] * 8) + (4 * e if case["bias"] else 0), "flops": 4 * rows * e}
    if kind == "quantize":
        return {"bytes": rows * case["in"] * (size + 1) + rows * case["in"] // GROUP * 4, "flops": 3 * rows * case["in"]}
    if kind == "linear":
        i, o = case["in"], case["out"]
        x = rows * i + rows * i // GROUP * 4 if case["given"] else rows * i * size
        return {"bytes": i * o + i // GROUP * -(-o // GROUP) * 4 + x + rows * o * size, "flops": 2 * rows * i * o}
    h, i, e, k = case["hidden"], case["inter"], case["experts"], case["topk"]
    chosen = k / (e * case["share"])  # how likely a row's k slots include a given expert
    used = e * (1.0 - (1.0 - chosen) ** rows)
    return {"bytes": used * (3 * h * i * (1 + 4 / GROUP ** 2)) + 2 * rows * h * size + rows * k * 8, "flops": 2 * rows * k / case["share"] * 3 * h * i}


def _e4m3(v):
    """64-bit values to the nearest e4m3 ones (ties to even), from the format: 3 mantissa bits, normal from 2^-6, at most 448."""
    exponent = torch.frexp(v)[1].to(torch.float64) - 1.0
    step = torch.exp2(exponent.clamp_min(-6.0) - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_values(x):
    groups = x.double().reshape(*x.shape[:-1], -1, GROUP)
    most = groups.abs().max(-1).values
    low = torch.exp2(torch.floor(torch.log2(most / 448.0)).clamp_min(-126.0) - 1.0)  # a logarithm next to a whole number may be off by a hair:
    times = (most > 448.0 * low).double() + (most > 896.0 * low) + (most > 1792.0 * low)  # the largest value itself decides
    scale = (low * torch.exp2(times)).clamp_min(2.0 ** -126)
    return _e4m3(groups / scale[..., None]), scale


def _exact_weight(w, scale):
    out, width = w.shape
    full = torch.zeros(scale.shape[0] * GROUP, width, dtype=torch.float64, device="cuda")
    full[:out] = w.double()
    full = full.reshape(scale.shape[0], GROUP, width // GROUP, GROUP) * scale.double()[:, None, :, None]
    return full.reshape(-1, width)[:out]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "route":
        x = state["logits"].double()
        if case["scoring"] == "softmax":
            e = torch.exp(x - x.max(-1, keepdim=True).values)
            score = e / e.sum(-1, keepdim=True)
        else:
            score = 1.0 / (1.0 + torch.exp(-x))
        pick = x.clone()
        if case["bias"] or case["groups"] > 1:
            pick = score + (0.0 if state["bias"] is None else state["bias"].double())
            wide = case["experts"] // case["groups"]
            sums = torch.stack([pick[:, g * wide : (g + 1) * wide].topk(min(2, wide)).values.sum(-1) for g in range(case["groups"])], -1)
            order = torch.argsort(-sums, dim=-1, stable=True)
            for place in range(case["group_topk"], case["groups"]):
                lost = order[:, place : place + 1] * wide + torch.arange(wide, device="cuda")
                pick.scatter_(-1, lost, -math.inf)
        inds = torch.argsort(-pick, dim=-1, stable=True)[:, : case["topk"]]
        chosen = torch.gather(score, -1, inds)
        if case["renormalise"]:
            chosen = chosen / chosen.sum(-1, keepdim=True)
        return inds.to(torch.int32), chosen * case["scale"]
    if case["kind"] == "quantize":
        q, scale = _exact_values(state["x"])
        return q.flatten(-2), scale
    if case["kind"] == "linear":
        q, scale = (state["q"].double().unflatten(-1, (-1, GROUP)), state["x_scale"].double()) if case["given"] else _exact_values(state["x"])
        return (q * scale[..., None]).flatten(-2) @ _exact_weight(state["w"], state["w_scale"]).T
    bank, inds, scores = state["bank"], state["inds"][0].tolist(), state["scores"][0].double()
    q, scale = _exact_values(state["x"][0])
    x = (q * scale[..., None]).flatten(-2)
    y = torch.zeros_like(x)
    for e in sorted({e for row in inds for e in row if e < case["experts"]}):
        gate, up, down = (_exact_weight(p.w[e], p.scale[e]) for p in (bank.gate, bank.up, bank.down))
        slots = [(r, k) for r, row in enumerate(inds) for k, v in enumerate(row) if v == e]
        at = torch.tensor([r for r, _ in slots], device="cuda")
        g = x[at] @ gate.T
        q, scale = _exact_values(g / (1.0 + torch.exp(-g)) * (x[at] @ up.T))
        y.index_add_(0, at, torch.stack([scores[r, k] for r, k in slots])[:, None] * ((q * scale[..., None]).flatten(-2) @ down.T))
    return y[None]
