"""The router on the device against its definition in 64 bits: choices equal, scores to a few 32-bit steps."""
import math

import pytest
import torch

import fp8_ref as ref
import turboexl3_b200 as t3

pytestmark = pytest.mark.gpu


def close(got, want):
    """exp is off by two steps, its argument's rounding by half a step of at most 2^7 (the logits' range here), the sums and divisions by one
    each of at most 40: 2 + 64 + 40 steps, taken for the chosen score and for the sum it is divided by."""
    got, want = got.double().cpu(), want
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    live = ~torch.isnan(want)
    assert torch.all((got - want)[live].abs() <= 212 * ref.STEP * want[live].abs() + 1e-37)


@pytest.mark.parametrize("rows,experts,topk,dtype,scoring,bias,groups,group_topk,renormalise,scale", [
    (1, 512, 10, torch.float32, "softmax", False, 1, 1, True, 1.0),
    (3, 1, 1, torch.float32, "softmax", False, 1, 1, True, 1.0),
    (5, 31, 31, torch.float32, "sigmoid", False, 1, 1, False, 1.0),
    (7, 33, 32, torch.float16, "softmax", False, 1, 1, True, 1.0),
    (129, 160, 6, torch.bfloat16, "softmax", False, 1, 1, False, 2.5),
    (33, 256, 8, torch.float32, "sigmoid", True, 8, 4, True, 2.5),
    (64, 1024, 32, torch.float32, "sigmoid", True, 32, 3, True, 1.0),
    (50, 1000, 5, torch.float32, "softmax", True, 1, 1, True, 1.0),
    (50, 513, 9, torch.bfloat16, "sigmoid", True, 27, 2, True, -1.5),
    (20, 64, 4, torch.float16, "softmax", False, 4, 1, True, 1.0),
    (20, 32, 3, torch.float32, "sigmoid", False, 32, 32, False, 1.0),
])
def test_choices_and_scores(rows, experts, topk, dtype, scoring, bias, groups, group_topk, renormalise, scale):
    gen = torch.Generator().manual_seed(rows * 1000 + experts)
    x = (torch.randn(rows, experts, generator=gen) * 2).to(dtype)
    b = 0.3 * torch.randn(experts, generator=gen) if bias else None
    inds, scores = t3.route(x.cuda(), topk, scoring, b.cuda() if bias else None, groups, group_topk, renormalise, scale)
    assert inds.dtype == torch.int32 and scores.dtype == torch.float32 and inds.shape == scores.shape == (rows, topk)
    want_i, want_s = ref.route(x, topk, scoring, b, groups, group_topk, renormalise, scale)
    assert torch.equal(inds.cpu().long(), want_i)
    close(scores, want_s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scoring,bias,groups", [("softmax", False, 1), ("sigmoid", False, 1), ("sigmoid", True, 1), ("sigmoid", True, 4), ("softmax", False, 4)])
def test_ties_masks_and_odd_values(dtype, scoring, bias, groups):
    low, inf, nan = torch.finfo(dtype).min, math.inf, math.nan
    n = 40
    rows = [[0.0] * n, [-0.0, 0.0] * (n // 2), [1.0, 2.0, 2.0, 1.0] * (n // 4), [low] * n, [-inf] * n, [low, -inf] * (n // 2),
            [low] * 17 + [0.5] + [low] * 22, [-inf] * 39 + [-3.0], [-90.0] * n, [0.0] * 20 + [-inf] * 20,
            [0.0] * 5 + [nan] + [1.0] * 34, [nan] * n]
    if scoring == "sigmoid":
        rows.append([inf] + [1.0] * 39)
    x = torch.tensor(rows, dtype=dtype)
    b = torch.linspace(-1, 1, 5).repeat(8) if bias else None
    got_i, got_s = t3.route(x.cuda(), 6, scoring, b.cuda() if bias else None, groups, min(2, groups), True, 1.0)
    want_i, want_s = ref.route(x, 6, scoring, b, groups, min(2, groups), True, 1.0)
    assert torch.equal(got_i.cpu().long(), want_i)
    close(got_s, want_s)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,group_topk,topk", [(64, 1, 1, 6), (64, 8, 3, 6), (8, 8, 5, 4), (60, 3, 2, 7), (1024, 2, 1, 16)])
def test_picks_that_32_bits_cannot_tell_apart(scoring, experts, groups, group_topk, topk):
    """Scores plus biases that differ by less than an f32 step of them, equal ones, and saturated scores: the order of the 64-bit sums."""
    gen = torch.Generator().manual_seed(experts + groups)
    x = torch.randint(-3, 4, (40, experts), generator=gen).float()
    x[10:20] += 2.0 ** -22 * torch.randint(-2, 3, (10, experts), generator=gen)
    x[20:25] = 30.0 + torch.randn(5, experts, generator=gen)
    x[25:30] = -torch.finfo(torch.float32).max
    x[27, ::5] = 1.0
    b = torch.randint(0, 3, (experts,), generator=gen).float() * 0.25 + 2.0 ** -24 * torch.randint(-1, 2, (experts,), generator=gen)
    got_i, got_s = t3.route(x.cuda(), topk, scoring, b.cuda(), groups, group_topk, True, 1.0)
    want_i, want_s = ref.route(x, topk, scoring, b, groups, group_topk, True, 1.0)
    assert torch.equal(got_i.cpu().long(), want_i)
    close(got_s, want_s)


def test_an_odd_bias_shows():
    x = torch.randn(4, 32, generator=torch.Generator().manual_seed(1))
    b = torch.zeros(32)
    b[7], b[9], b[11] = math.nan, math.inf, -math.inf
    for groups in (1, 4):
        got_i, _ = t3.route(x.cuda(), 3, "sigmoid", b.cuda(), groups, min(groups, 2))
        want_i, _ = ref.route(x, 3, "sigmoid", b, groups, min(groups, 2))
        assert torch.equal(got_i.cpu().long(), want_i)


def test_leading_shape_feeds_the_routed_layer():
    x = torch.randn(2, 3, 64, device="cuda")
    inds, scores = t3.route(x, 4)
    assert inds.shape == scores.shape == (2, 3, 4)
    flat = t3.route(x.view(6, 64), 4)
    assert torch.equal(inds.view(6, 4), flat[0]) and torch.equal(scores.view(6, 4), flat[1])


def test_a_captured_call_replays_on_new_logits():
    x = torch.randn(9, 96, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        t3.route(x, 5)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        inds, scores = t3.route(x, 5)
    for seed in (1, 2):
        x.copy_(torch.randn(9, 96, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        eager = t3.route(x, 5)
        torch.cuda.synchronize()
        assert torch.equal(inds, eager[0]) and torch.equal(scores, eager[1])


def test_python_refusals():
    x = torch.randn(2, 64, device="cuda")
    for call in (lambda: t3.route(x, 0), lambda: t3.route(x, 33), lambda: t3.route(x, 65), lambda: t3.route(x, 4, groups=5), lambda: t3.route(x[:0], 4),
                 lambda: t3.route(x, 4, bias=torch.zeros(63, device="cuda")), lambda: t3.route(x, 4, scale=math.inf)):
        with pytest.raises(t3.Exl3Error, match="BadExl3Shape"):
            call()
    for call in (lambda: t3.route(x.double(), 4), lambda: t3.route(x, 4, bias=torch.zeros(64, device="cuda", dtype=torch.float16))):
        with pytest.raises(t3.Exl3Error, match="BadExl3Dtype"):
            call()
    with pytest.raises(RuntimeError, match="contiguous"):
        t3.route(x.t(), 2)


def biased_rows(experts, seed, dtype=torch.float32):
    """Ordinary rows, rows that differ in their last bits, equal ones, and rows with removed experts."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(24, experts, generator=gen) * 2
    x[6:12] = torch.randint(-2, 3, (6, experts), generator=gen).float()
    x[9:12] += 2.0 ** -22 * torch.randint(-2, 3, (3, experts), generator=gen)
    x[12:18] = torch.where(torch.rand(6, experts, generator=gen) < 0.5, -math.inf, x[12:18])
    x[18:20] = torch.finfo(dtype).min
    x[20] = 0.0
    return x.to(dtype)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("experts,groups,group_topk,topk", [(8, 1, 1, 4), (4, 1, 1, 4), (64, 1, 1, 6), (160, 1, 1, 32), (8, 4, 2, 3), (16, 8, 3, 5),
                                                            (6, 3, 2, 4), (64, 8, 4, 8), (256, 8, 4, 8), (32, 32, 7, 7), (1024, 16, 5, 20)])
def test_a_bias_of_minus_infinity_puts_an_expert_last_and_removes_none(scoring, dtype, experts, groups, group_topk, topk):
    """Its pick is the lowest number there is; the expert is live: behind every other live one, ahead of a removed one, with its own score, and in its
    group's sum of two. A few finite biases, one, none; one -inf a group of two."""
    x = biased_rows(experts, experts + groups, dtype)
    gen = torch.Generator().manual_seed(groups)
    some = 0.25 * torch.randint(-1, 2, (experts,), generator=gen).float()
    for finite in (0, 1, 2, topk - 1, topk, topk + 1, experts - experts // 4, experts):
        b = torch.full((experts,), -math.inf)
        keep = torch.randperm(experts, generator=gen)[: min(finite, experts)]
        b[keep] = some[keep]
        got_i, got_s = t3.route(x.cuda(), topk, scoring, b.cuda(), groups, group_topk, True, 1.0)
        want_i, want_s = ref.route(x, topk, scoring, b, groups, group_topk, True, 1.0)
        assert torch.equal(got_i.cpu().long(), want_i), (finite, (got_i.cpu() != want_i).any(-1).nonzero().view(-1).tolist())
        close(got_s, want_s)


@pytest.mark.parametrize("scoring,bias", [("sigmoid", False), ("sigmoid", True), ("softmax", True)])
@pytest.mark.parametrize("groups", [1, 4])
def test_renormalised_scores_of_chosen_experts_far_below_one(scoring, bias, groups):
    """Scores that 32 bits hold with few bits or not at all still have a ratio: sigmoids of logits far below zero, and softmax's of experts that a
    bias chose far below the largest logit."""
    gen = torch.Generator().manual_seed(groups)
    n = 64
    x = torch.stack([shift + torch.randn(n, generator=gen) for shift in (-60.0, -80.0, -87.0, -92.0, -100.0, -104.0, -150.0, -600.0)])
    x[5, ::2] = -math.inf
    b = torch.zeros(n)
    if scoring == "softmax":
        x[:, 3] = 0.0  # takes all of the softmax, and is chosen last
        b[3] = -9.0
    if bias:
        b[10:40:3] += 0.5
    got_i, got_s = t3.route(x.cuda(), 5, scoring, b.cuda() if bias else None, groups, max(1, groups // 2), True, 2.5)
    want_i, want_s = ref.route(x, 5, scoring, b if bias else None, groups, max(1, groups // 2), True, 2.5)
    assert torch.equal(got_i.cpu().long(), want_i)
    assert torch.all(got_s.sum(-1).cpu() > 2.49)
    close(got_s, want_s)
