"""The 8-bit operators and the router in 64 bits, from their definitions, for the tests: plain loops over what they choose, no code of
the package. Errors allowed are counted from the roundings: a 32-bit step is 2^-23 relative (a sum of matrix products may cut instead of
round), an output's rounding half a step of its type."""
import math

import torch

GROUP = 128
STEP = 2.0 ** -23
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
LOWEST = {t: torch.finfo(t).min for t in HALF_STEP}


def power_of_two(e):
    """2^e in float64, exactly, for whole e in the normal range."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def e4m3_step(v):
    """The distance of neighbouring e4m3 values at |v| (float64)."""
    return power_of_two((torch.frexp(v.abs())[1] - 1).clamp_min(-6) - 3)


def e4m3(v):
    s = e4m3_step(v)
    return (torch.round(v / s) * s).clamp(-448.0, 448.0)


def quantize(x):
    """(values [..., in], scales [..., in / 128]) of x in float64: the smallest power of two with amax / scale <= 448."""
    g = x.double().unflatten(-1, (-1, GROUP))
    most = g.abs().amax(-1)
    bad = ~torch.isfinite(most)
    m, e = torch.frexp(torch.where(bad, 1.0, most).clamp_min(2.0 ** -140))
    scale = power_of_two((e - 9 + (m > 0.875)).clamp_min(-126))
    q = e4m3(g / scale[..., None])
    q = torch.where(bad[..., None], math.nan, q)
    return q.flatten(-2), torch.where(bad, math.nan, scale)


def weight(w, scale):
    """e4m3 [out, in] with a scale a 128 x 128 block, in float64."""
    full = scale.double().repeat_interleave(GROUP, 0)[: w.shape[0]].repeat_interleave(GROUP, 1)
    return w.double() * full


def linear(q, scale, w, w_scale):
    """(y, bound of its error ahead of the output's rounding)."""
    x, wd = q * scale.repeat_interleave(GROUP, -1), weight(w, w_scale)
    terms = GROUP + w.shape[1] // GROUP + 4
    return x @ wd.T, terms * STEP * (x.abs() @ wd.abs().T)


def out_bound(y, err, dtype):
    return err + HALF_STEP[dtype] * (y.abs() + err) + TINY[dtype]


def moe(x, gate, up, down, inds, scores, shared=None):
    """(y, bound) of the routed layer; gate, up, down = (w [E, out, in], scale), inds / scores [rows, topk]. What the second
    quantising may add: a value whose rounding lies within the error of its input may go to the neighbour."""
    q, s = quantize(x)
    rows, hidden = x.shape
    y = torch.zeros(rows, hidden, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(y)
    experts = gate[0].shape[0]
    for r in range(rows):
        for k in range(inds.shape[1]):
            e = int(inds[r, k])
            if e < 0 or e >= experts:
                continue
            g, dg = linear(q[r], s[r], gate[0][e], gate[1][e])
            u, du = linear(q[r], s[r], up[0][e], up[1][e])
            silu = g / (1.0 + torch.exp(-g))
            h = silu * u
            dh = 1.1 * dg * (u.abs() + du) + silu.abs() * du + 8 * STEP * h.abs()
            hq, hs = quantize(h)
            hs_full = hs.repeat_interleave(GROUP, -1)
            v = h / hs_full
            step = e4m3_step(v)
            off = (v / step - torch.floor(v / step) - 0.5).abs() * step  # from the border between two values
            near = off <= dh / hs_full
            # a group whose largest magnitude lies within its error of a power of two times 448 may take the next scale: its
            # smallest values then round to coarser steps
            most = h.unflatten(-1, (-1, GROUP)).abs().amax(-1)
            slack = dh.unflatten(-1, (-1, GROUP)).amax(-1)
            edge = ((most - 448.0 * hs).abs() <= slack) | ((most - 224.0 * hs).abs() <= slack)
            dq = torch.where(near, step, 0.0) + torch.where(edge.repeat_interleave(GROUP, -1), 2.0 ** -8, 0.0)
            d, dd = linear(hq, hs, down[0][e], down[1][e])
            dd = dd + (dq * hs_full) @ weight(down[0][e], down[1][e]).abs().T
            c = float(scores[r, k])
            y[r] += c * d
            err[r] += abs(c) * (dd + 8 * STEP * d.abs())
    if shared is not None:
        y = y + shared.double()
    return y, err + inds.shape[1] * STEP * y.abs()


def route(logits, topk, scoring, bias=None, groups=1, group_topk=1, renormalise=True, scale=1.0):
    """Lists a row: (experts, scores), from the definition, in Python's float64."""
    low = LOWEST[logits.dtype]
    chosen, scored = [], []
    for row in logits.double().tolist():
        live = [not v <= low for v in row]  # a NaN is live
        top = max((v for v, a in zip(row, live) if a and not math.isnan(v)), default=-math.inf)
        if scoring == "softmax":
            e = [(math.nan if math.isnan(v) or top == math.inf else math.exp(v - top)) if a else 0.0 for v, a in zip(row, live)]
            total = sum(e)
            score = [v / total if total else 0.0 for v in e]
        else:
            score = [(v if math.isnan(v) else 1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0) if a else 0.0 for v, a in zip(row, live)]
        pick = list(row)
        if bias is not None or groups > 1:
            pick = [s + (float(bias[i]) if bias is not None else 0.0) for i, s in enumerate(score)]
        key = [(2, 0.0) if a and math.isnan(p) else (1, p) if a else (0, 0.0) for p, a in zip(pick, live)]  # NaN first, the removed last
        inside = range(len(row))
        if groups > 1:
            wide = len(row) // groups
            ranks = []
            for g in range(groups):
                two = sorted((key[i] for i in range(g * wide, (g + 1) * wide) if live[i]), reverse=True)[:2]
                rank = (2, 0.0) if any(k[0] == 2 for k in two) else (1, sum(k[1] for k in two)) if two else (0, 0.0)
                ranks.append((rank, -g))
            keep = sorted(range(groups), key=lambda g: ranks[g], reverse=True)[:group_topk]
            inside = [i for i in inside if i // wide in keep]
        order = sorted(inside, key=lambda i: (key[i], -i), reverse=True)[:topk]
        s = [score[i] if live[i] else 0.0 for i in order]
        if renormalise:
            total = sum(s)
            s = [v / total if total else (v if math.isnan(total) else 0.0) for v in s]
        chosen.append(order)
        scored.append([v * scale for v in s])
    return torch.tensor(chosen), torch.tensor(scored, dtype=torch.float64)
