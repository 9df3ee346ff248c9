"""The 8-bit operators on the device against their definitions in 64 bits (fp8_ref): quantising to the bit, products within the counted
roundings."""
import math

import pytest
import torch

import fp8_ref as ref
import turboexl3_b200 as t3
from fp8_shapes import GEMM

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def activations(rows, width, dtype, seed, like=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = like * torch.randn(rows, width, generator=gen, device="cuda")
    x[:, ::37] *= 15.0
    return x.to(dtype)


def weights(shape, seed):
    """e4m3 values that fill the type's range (subnormals and both zeros among them) and a scale a block."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(shape, generator=gen, device="cuda") * 100).clamp_(-448, 448).to(E4M3)
    w.view(torch.uint8).view(-1)[::101] = 0x80
    w.view(torch.uint8).view(-1)[::103] = 0x03
    blocks = shape[:-2] + (-(-shape[-2] // 128), shape[-1] // 128)
    return w, (0.3 + torch.rand(blocks, generator=gen, device="cuda")) / (100.0 * math.sqrt(shape[-1]))


def held(got, want, bound):
    d = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    assert torch.all(d <= bound), (float(d.max()), float((d / bound).max()), int((d > bound).sum()))


# ---- quantising ----

@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(1, 128), (1, 7168), (3, 384), (37, 2048), (1111, 256)])
def test_quantize_is_the_definitions(rows, width, dtype):
    x = activations(rows, width, dtype, rows + width)
    q, s = t3.quantize_fp8(x)
    want_q, want_s = ref.quantize(x)
    assert q.dtype == E4M3 and q.shape == x.shape and s.shape == (rows, width // 128)
    assert torch.equal(s.double(), want_s)
    assert torch.equal(q.double(), want_q)


def test_quantize_at_the_edges():
    rows = [[0.0], [448.0], [449.0], [-448.0, 447.9], [464.0], [2.0 ** -126 * 448], [2.0 ** -149], [2.0 ** -120, -(2.0 ** -149)], [3.4e38, 1.0], [1e30, 1e24, 1.5e27],
            [1.75, 1.0625, 1.1875, 0.0625 * 1.0625, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -10], [1.7500001], [-0.0, 1.0], [448.0 * 2.0 ** 119]]
    x = torch.zeros(len(rows), 128)
    for i, r in enumerate(rows):
        x[i, : len(r)] = torch.tensor(r)
    q, s = t3.quantize_fp8(x.cuda())
    want_q, want_s = ref.quantize(x)
    assert torch.equal(s.double().cpu(), want_s)
    assert torch.equal(q.cpu().double(), want_q)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_quantize_of_an_infinity_or_nan_is_its_groups_alone(bad):
    x = activations(4, 512, torch.bfloat16, 5)
    x[2, 200] = bad
    q, s = t3.quantize_fp8(x)
    want_q, want_s = ref.quantize(x)
    assert torch.isnan(s[2, 1]) and torch.isnan(q[2, 128:256].float()).all()
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(want_s.cpu()))
    assert torch.equal(q.double().nan_to_num(9e9), want_q.nan_to_num(9e9))


# ---- the linear ----

@pytest.mark.parametrize("rows,width,out,dtype", [
    (1, 128, 1, torch.bfloat16), (1, 2048, 2048, torch.bfloat16), (1, 131072, 128, torch.bfloat16), (2, 256, 17, torch.float16), (7, 1536, 576, torch.float32),
    (16, 640, 255, torch.bfloat16), (17, 1024, 384, torch.float16), (29, 16384, 256, torch.bfloat16), (32, 384, 4096, torch.float32),
    (33, 512, 130, torch.bfloat16), (64, 2048, 128, torch.float16), (65, 896, 640, torch.float32), (128, 256, 1000, torch.bfloat16),
    (129, 7168, 576, torch.bfloat16), (300, 640, 333, torch.float32), (1000, 384, 1408, torch.float16), (2050, 128, 2048, torch.bfloat16),
    (2500, 640, 2309, torch.float16), (1100, 1664, 4100, torch.float32), (257, 1024, 20001, torch.bfloat16),
])
def test_linear_against_64_bits(rows, width, out, dtype):
    x = activations(rows, width, dtype, rows)
    w, ws = weights((out, width), out)
    y = t3.linear_fp8(x, w, ws)
    assert y.shape == (rows, out) and y.dtype == dtype
    q, s = ref.quantize(x)
    want, err = ref.linear(q, s, w, ws)
    held(y, want, ref.out_bound(want, err, dtype))
    # its own quantised rows give the same bytes
    given = t3.linear_fp8(*[t3.quantize_fp8(x)[0], w, ws], x_scale=t3.quantize_fp8(x)[1], out_dtype=dtype)
    assert torch.equal(given, y)
    assert t3.device_error() == 0


@pytest.mark.parametrize("rows", [1, 20, 40, 150])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_linear_takes_any_scales(rows, out_dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = activations(rows, 512, torch.float32, rows, 100.0).clamp(-448, 448).to(E4M3)
    s = torch.rand(rows, 4, generator=gen, device="cuda") * 0.01 - 0.003
    w, ws = weights((200, 512), rows + 1)
    want, err = ref.linear(x.double(), s.double(), w, ws)
    held(t3.linear_fp8(x, w, ws, s, out_dtype), want, ref.out_bound(want, err, out_dtype))


def test_linear_rows_with_a_nan_leave_the_others():
    for rows, bad in ((5, 3), (31, 30), (60, 59), (200, 130)):
        x = activations(rows, 256, torch.bfloat16, rows)
        w, ws = weights((300, 256), 9)
        clean = t3.linear_fp8(x, w, ws)
        x[bad, 7] = math.nan
        y = t3.linear_fp8(x, w, ws)
        keep = torch.arange(rows) != bad
        assert torch.isnan(y[bad].float()).all() and torch.equal(y[keep], clean[keep])


def test_linear_of_a_nan_weight_is_that_output_alone():
    x = activations(3, 256, torch.bfloat16, 1)
    w, ws = weights((300, 256), 2)
    clean = t3.linear_fp8(x, w, ws)
    w.view(torch.uint8)[129, 200] = 0x7F
    y = t3.linear_fp8(x, w, ws)
    keep = torch.arange(300) != 129
    assert torch.isnan(y[:, 129].float()).all() and torch.equal(y[:, keep], clean[:, keep])


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_linear_writes_its_rows_and_nothing_else(rows):
    """The call on a buffer with room around it (through the C ABI): the bytes before and behind stay."""
    width, out = 256, 131
    x = activations(rows, width, torch.bfloat16, 3)
    w, ws = weights((out, width), 4)
    room = torch.full((rows * out + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    L = t3.lib()
    need = L.t3_linear_fp8_workspace_bytes(rows, width, out, 2)
    work = torch.full((need + 512,), 0x55, dtype=torch.uint8, device="cuda")
    at = room[32:]
    assert at.data_ptr() % 16 == 0
    assert L.t3_linear_fp8(x.data_ptr(), 2, None, rows, w.data_ptr(), ws.data_ptr(), width, out, at.data_ptr(), 2, work.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.all(room[:32] == 7) and torch.all(room[32 + rows * out:] == 7) and torch.all(work[need:] == 0x55)
    assert torch.equal(at[: rows * out].view(rows, out), t3.linear_fp8(x, w, ws))


# ---- the routed layer ----

def bank(experts, hidden, inter, seed):
    p = [weights((experts, o, i), seed + n) for n, (o, i) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    return t3.Fp8Bank(*[t3.Fp8Proj(w, s) for w, s in p]), p


def check_moe(x, b, parts, inds, scores, shared=None):
    y = t3.moe_fp8(x[None], b, inds[None], scores[None], None if shared is None else shared[None])[0]
    want, err = ref.moe(x, *parts, inds.long(), scores, shared)
    held(y, want, ref.out_bound(want, err, x.dtype))
    assert t3.device_error() == 0
    return y


@pytest.mark.parametrize("rows,hidden,inter,experts,topk,dtype", [
    (1, 128, 128, 1, 1, torch.bfloat16), (1, 2048, 512, 64, 10, torch.bfloat16), (2, 384, 256, 5, 3, torch.float16), (4, 640, 128, 33, 4, torch.float32),
    (16, 256, 384, 16, 2, torch.bfloat16), (17, 1024, 256, 9, 3, torch.float16), (32, 512, 640, 40, 8, torch.bfloat16), (9, 7168, 256, 6, 2, torch.bfloat16),
    (32, 7168, 128, 4, 1, torch.float16), (3, 256, 2048, 7, 7, torch.bfloat16),
])
def test_moe_against_64_bits(rows, hidden, inter, experts, topk, dtype):
    x = activations(rows, hidden, dtype, rows)
    b, parts = bank(experts, hidden, inter, 11)
    logits = torch.randn(rows, experts, generator=torch.Generator().manual_seed(rows)).cuda()
    inds, scores = t3.route(logits, topk)
    check_moe(x, b, parts, inds, scores)


def test_moe_ids_elsewhere_and_twice():
    x = activations(6, 256, torch.bfloat16, 1)
    b, parts = bank(8, 256, 256, 21)
    inds = torch.tensor([[0, 1, 2], [8, 9, -1], [3, 3, 3], [7, 100, 7], [-(2 ** 31), 2 ** 31 - 1, 0], [5, 8, 6]], dtype=torch.int32, device="cuda")
    scores = torch.rand(6, 3, device="cuda") + 0.1
    scores[1] = math.nan  # a padded row's: nobody's
    scores[5, 1] = math.inf
    y = check_moe(x, b, parts, inds, scores)
    assert torch.all(y[1] == 0)
    shared = activations(6, 256, torch.bfloat16, 2)
    y = check_moe(x, b, parts, inds, scores, shared)
    assert torch.equal(y[1], shared[1])


@pytest.mark.parametrize("rows", [1, 16, 32])
def test_moe_with_no_expert_here_is_the_shared_one(rows):
    x = activations(rows, 256, torch.float16, 1)
    b, _ = bank(4, 256, 128, 3)
    inds = torch.full((1, rows, 2), 4, dtype=torch.int32, device="cuda")
    scores = torch.ones(1, rows, 2, device="cuda")
    assert torch.all(t3.moe_fp8(x[None], b, inds, scores) == 0)
    assert torch.equal(t3.moe_fp8(x[None], b, inds, scores, x[None])[0], x)


@pytest.mark.parametrize("scores_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_moe_every_row_to_one_expert(scores_dtype):
    x = activations(32, 384, torch.bfloat16, 8)
    b, parts = bank(3, 384, 128, 5)
    inds = torch.full((32, 2), 2, dtype=torch.uint32, device="cuda")
    scores = torch.rand(32, 2, device="cuda").to(scores_dtype)
    y = check_moe(x, b, parts, inds.to(torch.int32), scores.float())
    assert torch.equal(t3.moe_fp8(x[None], b, inds[None], scores[None])[0], y) or scores_dtype != torch.float32


def test_moe_a_nan_row_leaves_the_others():
    x = activations(20, 512, torch.bfloat16, 8)
    b, parts = bank(6, 512, 256, 5)
    inds, scores = t3.route(torch.randn(20, 6, device="cuda"), 2)
    clean = check_moe(x, b, parts, inds, scores)
    x[11, 3] = math.inf
    y = t3.moe_fp8(x[None], b, inds[None], scores[None])[0]
    keep = torch.arange(20) != 11
    assert torch.isnan(y[11].float()).all() and torch.equal(y[keep], clean[keep])


def test_moe_a_nan_expert_is_its_rows_alone():
    x = activations(9, 256, torch.bfloat16, 8)
    b, parts = bank(6, 256, 256, 5)
    inds = torch.tensor([[i % 5, 5 if i in (2, 7) else (i + 1) % 5] for i in range(9)], dtype=torch.int32, device="cuda")
    scores = torch.rand(9, 2, device="cuda")
    clean = check_moe(x, b, parts, inds, scores)
    b.down.w.view(torch.uint8)[5, 7, :] = 0x7F
    b.up.scale[5, 1, 0] = math.nan
    b.down.scale[5, 0, 0] = math.inf
    y = t3.moe_fp8(x[None], b, inds[None], scores[None])[0]
    keep = torch.tensor([i not in (2, 7) for i in range(9)])
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[~keep].float()).all()


def test_moe_batch_shape_and_refusals():
    b, _ = bank(4, 256, 128, 3)
    x = activations(6, 256, torch.bfloat16, 1).view(2, 3, 256)
    inds = torch.randint(0, 4, (2, 3, 2), device="cuda", dtype=torch.int32)
    scores = torch.rand(2, 3, 2, device="cuda")
    y = t3.moe_fp8(x, b, inds, scores)
    assert y.shape == x.shape
    assert torch.equal(y.view(1, 6, 256), t3.moe_fp8(x.view(1, 6, 256), b, inds.view(1, 6, 2), scores.view(1, 6, 2)))
    with pytest.raises(t3.Exl3Error, match="Exl3EngineNotImplemented"):
        t3.moe_fp8(x.repeat(1, 11, 1), b, inds.repeat(1, 11, 1), scores.repeat(1, 11, 1))
    with pytest.raises(t3.Exl3Error, match="BadExl3Dtype"):
        t3.moe_fp8(x, b, inds.long(), scores)
    with pytest.raises(t3.Exl3Error, match="BadExl3Shape"):
        t3.moe_fp8(x[..., :128].contiguous(), b, inds, scores)
    with pytest.raises(RuntimeError, match="contiguous"):
        t3.moe_fp8(x.transpose(0, 1), b, inds.transpose(0, 1), scores.transpose(0, 1))


def test_linear_refusals():
    w, ws = weights((200, 256), 1)
    x = activations(3, 256, torch.bfloat16, 1)
    q, s = t3.quantize_fp8(x)
    cases = [(lambda: t3.linear_fp8(x[:, :128].contiguous(), w, ws), "BadExl3Shape"), (lambda: t3.linear_fp8(x, w, ws[:1].contiguous()), "BadExl3Shape"),
             (lambda: t3.linear_fp8(x[:0], w, ws), "BadExl3Shape"), (lambda: t3.linear_fp8(x, w, ws, s), "BadExl3Shape"),
             (lambda: t3.linear_fp8(q, w, ws, s[:2].contiguous()), "BadExl3Shape"), (lambda: t3.linear_fp8(q, w, ws), "NullPointer"),
             (lambda: t3.linear_fp8(x.double(), w, ws), "BadExl3Dtype"), (lambda: t3.linear_fp8(x, w.view(torch.uint8), ws), "BadExl3Dtype"),
             (lambda: t3.linear_fp8(x, w, ws.half()), "BadExl3Dtype"), (lambda: t3.linear_fp8(x.view(-1)[8:8 + 256 + 256].view(2, 256)[:, :], w, ws), None),
             (lambda: t3.linear_fp8(x.view(-1)[4:4 + 512].view(2, 256), w, ws), "BadExl3Shape"),
             (lambda: t3.quantize_fp8(x.view(-1)[:200].view(1, 200)), "BadExl3Shape"), (lambda: t3.quantize_fp8(x.double()), "BadExl3Dtype"),
             (lambda: t3.quantize_fp8(x.view(-1)[1:129].view(1, 128)), "BadExl3Shape")]
    for call, why in cases:
        if why is None:
            call()
            continue
        with pytest.raises(t3.Exl3Error, match=why):
            call()


# ---- as they are used together ----

def test_a_layer_of_both_kinds_in_a_graph_and_on_another_stream():
    """Logits by an 8-bit linear, the routing, an 8-bit routed layer and an 8-bit projection of its output: eager, on a side stream, captured and
    replayed on new rows give the same bytes."""
    rows, hidden, experts = 5, 512, 24
    b, _ = bank(experts, hidden, 256, 31)
    gate = weights((experts, hidden), 41)
    proj = weights((700, hidden), 42)

    def layer(x):
        inds, scores = t3.route(t3.linear_fp8(x, *gate), 4, "sigmoid", scale=2.5)
        y = t3.moe_fp8(x, b, inds, scores)
        q, s = t3.quantize_fp8(y)
        return t3.linear_fp8(q, *proj, x_scale=s), y

    x = activations(rows, hidden, torch.bfloat16, 1).view(1, rows, hidden)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x)
    torch.cuda.current_stream().wait_stream(side)
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer(x)
    with torch.cuda.graph(g2):
        out2 = layer(x)
    for seed in range(3):
        x.copy_(activations(rows, hidden, torch.bfloat16, 50 + seed).view_as(x))
        eager = layer(x)
        g.replay()
        g2.replay()
        g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = layer(x)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for got in (out, out2, other):
            assert all(torch.equal(a, e) for a, e in zip(got, eager))
    assert t3.device_error() == 0


def test_two_streams_at_once():
    b, _ = bank(16, 512, 256, 31)
    w, ws = weights((1024, 512), 4)
    xs = [activations(9, 512, torch.bfloat16, 60 + i).view(1, 9, 512) for i in range(2)]
    route = [t3.route(torch.randn(1, 9, 16, device="cuda"), 3) for _ in xs]
    want = [(t3.moe_fp8(x, b, *r), t3.linear_fp8(x, w, ws)) for x, r in zip(xs, route)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((t3.moe_fp8(xs[i], b, *route[i]), t3.linear_fp8(xs[i], w, ws)))
    torch.cuda.synchronize()
    for i in range(2):
        for m, l in got[i]:
            assert torch.equal(m, want[i][0]) and torch.equal(l, want[i][1])
    assert t3.device_error() == 0


def test_without_launch_overlap_the_bytes_are_the_same():
    b, _ = bank(12, 384, 256, 31)
    x = activations(8, 384, torch.float16, 3).view(1, 8, 384)
    r = t3.route(torch.randn(1, 8, 12, device="cuda"), 3)
    w, ws = weights((300, 384), 4)
    want = t3.moe_fp8(x, b, *r), t3.linear_fp8(x, w, ws)
    t3.configure(no_overlap=True)
    try:
        assert torch.equal(t3.moe_fp8(x, b, *r), want[0]) and torch.equal(t3.linear_fp8(x, w, ws), want[1])
    finally:
        t3.configure()


def test_the_exl3_layer_takes_the_same_routing():
    rows, hidden, inter, experts = 3, 256, 128, 8
    gen = torch.Generator(device="cuda").manual_seed(1)

    def proj(i, o):
        return t3.Proj(torch.randint(-32768, 32768, (experts, i // 16, o // 16, 64), generator=gen, device="cuda", dtype=torch.int16),
                       torch.full((experts, i), 2.0 ** -4, device="cuda", dtype=torch.float16), torch.ones(experts, o, device="cuda", dtype=torch.float16))

    exl3 = t3.Bank(proj(hidden, inter), proj(hidden, inter), proj(inter, hidden))
    x = torch.randn(1, rows, hidden, generator=gen, device="cuda").half()
    inds, scores = t3.route(torch.randn(1, rows, experts, generator=gen, device="cuda"), 2)
    y = t3.moe(x, exl3, inds, scores)
    want = sum(scores[..., k:k + 1] * t3.moe(x, exl3, inds[..., k:k + 1].contiguous(), torch.ones_like(scores[..., :1])).float() for k in range(2))
    # the two experts' outputs are rounded to 16 bits once more here than in the layer, and so is their sum
    assert torch.all((y.float() - want).abs() <= 4 * 2.0 ** -11 * (want.abs() + y.float().abs().amax()))


@pytest.mark.parametrize("rows,hidden,inter,experts,topk", [(12, 512, 2048, 64, 9), (3, 640, 1792, 46, 8), (32, 1024, 512, 8, 2), (1, 384, 256, 30, 5)])
def test_calls_behind_one_another_leave_each_other_alone(rows, hidden, inter, experts, topk):
    """Many calls in a row, each launch starting while the one before it ends: every one gives the first one's bytes."""
    b, _ = bank(experts, hidden, inter, 71)
    x = activations(rows, hidden, torch.bfloat16, 4).view(1, rows, hidden)
    r = t3.route(torch.randn(1, rows, experts, generator=torch.Generator("cuda").manual_seed(1), device="cuda"), topk)
    w, ws = weights((1100, hidden), 5)
    first = t3.moe_fp8(x, b, *r), t3.linear_fp8(x, w, ws)
    got = [(t3.moe_fp8(x, b, *r), t3.linear_fp8(x, w, ws)) for _ in range(200)]
    torch.cuda.synchronize()
    assert all(torch.equal(m, first[0]) and torch.equal(l, first[1]) for m, l in got)
    assert t3.device_error() == 0


@pytest.mark.parametrize("rows,width,out", [(1, 2048, 384), (20, 4096, 640), (40, 7168, 130), (200, 7168, 576), (300, 256, 1000)])
def test_linears_behind_one_another_leave_each_other_alone(rows, width, out):
    x = activations(rows, width, torch.bfloat16, 6)
    w, ws = weights((out, width), 7)
    first = t3.linear_fp8(x, w, ws)
    got = [t3.linear_fp8(x, w, ws) for _ in range(200)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, first) for y in got)
    assert t3.device_error() == 0


def test_a_mix_on_four_streams():
    """Routed layers and linears of several shapes, EXL3 linears and routings, drawn at random onto four streams: each call gives the bytes it
    gives alone."""
    import random
    jobs = []

    def job(call):
        alone = call()
        torch.cuda.synchronize()
        jobs.append((call, alone))

    for rows, hidden, inter, experts, topk in ((12, 512, 1024, 32, 5), (1, 1024, 512, 64, 8), (29, 1024, 256, 64, 6), (32, 256, 512, 8, 2)):
        b, _ = bank(experts, hidden, inter, rows)
        x = activations(rows, hidden, torch.bfloat16, rows).view(1, rows, hidden)
        r = t3.route(torch.randn(1, rows, experts, device="cuda"), topk)
        job(lambda x=x, b=b, r=r: t3.moe_fp8(x, b, *r))
    for rows, width, out in ((1, 2048, 2048), (29, 8192, 512), (200, 7168, 576), (900, 512, 3001), (17, 512, 20000), (64, 4096, 300)):
        w, ws = weights((out, width), out)
        x = activations(rows, width, torch.float16, rows)
        job(lambda x=x, w=w, ws=ws: t3.linear_fp8(x, w, ws))
    trellis = torch.randint(-32768, 32768, (64, 64, 64), device="cuda", dtype=torch.int16)
    ones = torch.ones(1024, device="cuda", dtype=torch.float16)
    for rows in (1, 100):
        x = torch.randn(rows, 1024, device="cuda").half()
        job(lambda x=x: t3.linear(x, trellis, ones, ones))
    logits, bias = torch.randn(500, 256, device="cuda"), 0.1 * torch.randn(256, device="cuda")
    job(lambda: t3.route(logits, 8, "sigmoid", bias, 8, 4)[0])
    rng, streams = random.Random(1), [torch.cuda.Stream() for _ in range(4)]
    for _ in range(15):
        done = []
        for s in streams:
            with torch.cuda.stream(s):
                for _ in range(10):
                    call, alone = rng.choice(jobs)
                    done.append((call(), alone))
        torch.cuda.synchronize()
        assert all(torch.equal(y, alone) for y, alone in done)
    assert t3.device_error() == 0


# ---- where a tensor starts and how far it reaches ----

def test_scales_and_routing_on_their_own_types_alignment():
    """Only activations, e4m3 values and outputs have to start on 16 bytes."""
    def moved(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:] = t.reshape(-1)
        return room[1:].view(t.shape)
    for rows in (3, 31, 70):
        x = activations(rows, 640, torch.bfloat16, rows)
        w, ws = weights((200, 640), 2)
        q, s = t3.quantize_fp8(x)
        assert torch.equal(t3.linear_fp8(x, w, moved(ws)), t3.linear_fp8(x, w, ws))
        assert torch.equal(t3.linear_fp8(q, w, moved(ws), moved(s)), t3.linear_fp8(q, w, ws, s))
    b, _ = bank(6, 256, 384, 3)
    off = t3.Fp8Bank(*[t3.Fp8Proj(p.w, moved(p.scale)) for p in (b.gate, b.up, b.down)])
    x = activations(9, 256, torch.float16, 1).view(1, 9, 256)
    logits = torch.randn(1, 9, 6, device="cuda").bfloat16()
    bias = torch.rand(6, device="cuda")
    inds, scores = t3.route(logits, 3, "sigmoid", bias)
    got = t3.route(moved(logits), 3, "sigmoid", moved(bias))
    assert torch.equal(got[0], inds) and torch.equal(got[1], scores)
    assert torch.equal(t3.moe_fp8(x, off, moved(inds), moved(scores.half())), t3.moe_fp8(x, b, inds, scores.half()))
    assert t3.device_error() == 0


def test_quantize_past_32_bits():
    rows, width = 600000, 7168
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    x[-70:] = activations(70, width, torch.bfloat16, 1)
    q, s = t3.quantize_fp8(x)
    want_q, want_s = ref.quantize(x[-70:])
    assert torch.equal(q[-70:].double(), want_q) and torch.equal(s[-70:].double(), want_s)
    assert float(s[-71].max()) == 2.0 ** -126 and int(q[-71].view(torch.uint8).max()) == 0


@pytest.mark.parametrize("rows,width", [(1, 32768), (30, 32768), (40, 32768), (8000, 128)])
def test_linear_past_32_bits(rows, width):
    """Weights of more than 4 GiB, and outputs."""
    out, end = 1094 * 128, 384
    w = torch.zeros(out, width, dtype=torch.uint8, device="cuda").view(E4M3)
    ws = torch.ones(out // 128, width // 128, device="cuda")
    tail, tail_s = weights((end, width), 7)
    w.view(torch.uint8)[-end:] = tail.view(torch.uint8)
    ws[-end // 128:] = tail_s
    x = activations(rows, width, torch.bfloat16, rows)
    q, s = t3.quantize_fp8(x)
    y = t3.linear_fp8(q, w, ws, s, torch.float32)
    part = slice(max(0, rows - 200), rows)
    want, err = ref.linear(*ref.quantize(x[part]), tail, tail_s)
    held(y[part, -end:], want, ref.out_bound(want, err, torch.float32))
    assert int(torch.count_nonzero(y[:, :-end])) == 0
    assert t3.device_error() == 0


def test_moe_past_32_bits():
    experts, hidden, inter, end = 2048, 2048, 1152, 8
    small, parts = bank(end, hidden, inter, 5)

    def behind(p):
        w = torch.zeros((experts,) + p.w.shape[1:], dtype=torch.uint8, device="cuda")
        s = torch.ones((experts,) + p.scale.shape[1:], device="cuda")
        w[-end:], s[-end:] = p.w.view(torch.uint8), p.scale
        return t3.Fp8Proj(w.view(E4M3), s)
    big = t3.Fp8Bank(*[behind(p) for p in (small.gate, small.up, small.down)])
    for rows in (1, 4, 20):
        x = activations(rows, hidden, torch.bfloat16, rows).view(1, rows, hidden)
        inds = torch.randint(0, end, (1, rows, 2), device="cuda", dtype=torch.int32)
        scores = torch.rand(1, rows, 2, device="cuda")
        y = t3.moe_fp8(x, big, inds + (experts - end), scores)[0]
        want, err = ref.moe(x[0], *parts, inds[0].long(), scores[0])
        held(y, want, ref.out_bound(want, err, x.dtype))
    assert t3.device_error() == 0


@pytest.mark.parametrize("rows,width,out", [(20, 4096, 640), (40, 7168, 130), (200, 7168, 576), (300, 1024, 1000), (1500, 512, 2048)])
def test_linears_behind_one_another_read_their_own_rows_scales(rows, width, out):
    """Calls in a row, in a stream and in a graph, on rows that are another power of two times larger each: the quantised values are the same, at the
    same address of the workspace, and the scales alone differ. Every output is the first one's times that power, exactly."""
    x = activations(rows, width, torch.bfloat16, 6)
    w, ws = weights((out, width), 7)
    powers = [0, 3, -5, 11, -9, 1, 7, -2]
    xs = [x * 2.0 ** p for p in powers]
    first = t3.linear_fp8(x, w, ws, out_dtype=torch.float32)
    for _ in range(20):
        got = [t3.linear_fp8(v, w, ws, out_dtype=torch.float32) for v in xs]
        assert all(torch.equal(y, first * 2.0 ** p) for y, p in zip(got, powers))
    g = torch.cuda.CUDAGraph()
    moving = x.clone()
    with torch.cuda.graph(g):
        y = [t3.linear_fp8(moving, w, ws, out_dtype=torch.float32) for _ in range(3)]
    for v, p in zip(xs, powers):
        moving.copy_(v)
        g.replay()
        assert all(torch.equal(r, first * 2.0 ** p) for r in y)
    assert t3.device_error() == 0


@pytest.mark.parametrize("rows,topk", [(1, 4), (5, 3), (32, 8)])
def test_routings_behind_one_another_at_the_same_addresses(rows, topk):
    """Routings of changing logits, each ahead of both kinds of routed layer, which read the choice ahead of their second launch's own wait: a captured
    chain of three, replayed on new logits, whose outputs lie at the same addresses every time, gives the eager calls' bytes."""
    hidden, inter, experts = 256, 128, 48
    gen = torch.Generator(device="cuda").manual_seed(rows)

    def proj(i, o):
        return t3.Proj(torch.randint(-32768, 32768, (experts, i // 16, o // 16, 64), generator=gen, device="cuda", dtype=torch.int16),
                       torch.full((experts, i), 2.0 ** -4, device="cuda", dtype=torch.float16), torch.ones(experts, o, device="cuda", dtype=torch.float16))

    exl3 = t3.Bank(proj(hidden, inter), proj(hidden, inter), proj(inter, hidden))
    fp8, _ = bank(experts, hidden, inter, 51)
    x = activations(rows, hidden, torch.float16, 3).view(1, rows, hidden)
    logits = [torch.empty(1, rows, experts, device="cuda") for _ in range(3)]

    def chain():
        out = []
        for l in logits:
            inds, scores = t3.route(l, topk)
            out += [inds, scores, t3.moe(x, exl3, inds, scores), t3.moe_fp8(x, fp8, inds, scores)]
        return out

    def alone():
        out = []
        for l in logits:
            inds, scores = t3.route(l, topk)
            torch.cuda.synchronize()
            for layer, b in ((t3.moe, exl3), (t3.moe_fp8, fp8)):
                out.append(layer(x, b, inds, scores))
                torch.cuda.synchronize()
        return out

    for l in logits:
        l.normal_(generator=gen)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = chain()
    before = None
    for _ in range(12):
        for l in logits:
            l.normal_(generator=gen)
        g.replay()
        g.replay()
        eager = chain()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        assert all(torch.equal(a, b) for a, b in zip([v for i, v in enumerate(got) if i % 4 > 1], alone()))
        assert before is None or not torch.equal(before, got[0])  # (the choice did change)
        before = got[0].clone()
    assert t3.device_error() == 0


@pytest.mark.parametrize("scores_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,topk", [(3, 2), (16, 2), (32, 5)])
def test_moe_scores_in_16_bits_are_their_f32_values(scores_dtype, rows, topk):
    """Few slots and more than a warp's, against 64 bits and, to the byte, against the same scores held in f32."""
    x = activations(rows, 384, torch.bfloat16, 8)
    b, parts = bank(7, 384, 128, 5)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    inds = torch.randint(0, 7, (rows, topk), generator=gen, device="cuda", dtype=torch.int32)
    scores = (torch.rand(rows, topk, generator=gen, device="cuda") + 0.05).to(scores_dtype)
    y = check_moe(x, b, parts, inds, scores)
    assert torch.equal(y, t3.moe_fp8(x[None], b, inds[None], scores.float()[None])[0])
    # every row to one expert, its slots' scores added up
    one = torch.full((rows, topk), 2, dtype=torch.int32, device="cuda")
    y = check_moe(x, b, parts, one, scores)
    assert torch.equal(y, t3.moe_fp8(x[None], b, one[None].view(torch.uint32), scores.float()[None])[0])


@pytest.mark.parametrize("rows,width,out", sorted(GEMM))
def test_every_kernel_of_the_gemm(rows, width, out):
    """Against 64 bits, the three output types in turn; then calls behind one another, on two streams, give the first one's bytes."""
    dtype = (torch.bfloat16, torch.float16, torch.float32)[(rows + out) % 3]
    x = activations(rows, width, dtype, rows)
    w, ws = weights((out, width), out)
    y = t3.linear_fp8(x, w, ws)
    q, s = ref.quantize(x)
    want, err = ref.linear(q, s, w, ws)
    held(y, want, ref.out_bound(want, err, dtype))
    mine, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(mine)
    got = []
    for i in range(60):
        with torch.cuda.stream(side if i % 3 == 2 else mine):
            got.append(t3.linear_fp8(x, w, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(v, y) for v in got)
    assert t3.device_error() == 0


def test_the_exl3_records_are_the_exl3_calls_alone():
    """engines_held counts the geometries of EXL3 calls, as the reference's does; last_kernel_symbol names an EXL3 decode-row kernel."""
    trellis = torch.randint(-32768, 32768, (16, 16, 64), device="cuda", dtype=torch.int16)
    ones = torch.ones(256, device="cuda", dtype=torch.float16)
    t3.release_engines()
    t3.linear(torch.randn(1, 256, device="cuda").half(), trellis, ones, ones)
    held_before, symbol = t3.engines_held(), t3.last_kernel_symbol()
    assert held_before == {"decode": 0, "dense": 1, "prefill": 0}
    b, _ = bank(4, 256, 128, 3)
    w, ws = weights((256, 256), 1)
    for rows in (2, 100):
        t3.linear_fp8(activations(rows, 256, torch.bfloat16, 1), w, ws)
    x = activations(3, 256, torch.bfloat16, 1).view(1, 3, 256)
    t3.moe_fp8(x, b, *t3.route(torch.randn(1, 3, 4, device="cuda"), 2))
    t3.quantize_fp8(x)
    assert t3.engines_held() == held_before and t3.last_kernel_symbol() == symbol
    t3.release_engines()


@pytest.mark.parametrize("rows,hidden,inter,experts,topk", [(1, 4096, 2048, 8, 4), (1, 4096, 256, 128, 4), (2, 1024, 256, 2048, 2), (32, 512, 128, 128, 32)])
def test_moe_whose_down_takes_what_gate_and_up_leave(rows, hidden, inter, experts, topk):
    """Shapes whose second launch has its weights in flight cut to the shared memory that the first one's CTAs leave a multiprocessor."""
    x = activations(rows, hidden, torch.bfloat16, rows)
    b, parts = bank(experts, hidden, inter, 11)
    scores, inds = torch.randn(rows, experts, generator=torch.Generator().manual_seed(rows)).softmax(-1).cuda().topk(topk)  # (2048: more than route takes)
    inds = inds.to(torch.int32)
    y = check_moe(x, b, parts, inds, scores)
    got = [t3.moe_fp8(x[None], b, inds[None], scores[None])[0] for _ in range(50)]
    assert all(torch.equal(v, y) for v in got)
    assert t3.device_error() == 0


def test_a_wait_that_runs_out_is_reported_once_and_the_next_calls_run():
    assert t3.device_error() == 0
    w, ws = weights((256, 512), 1)
    x = activations(40, 512, torch.bfloat16, 1)
    want = t3.linear_fp8(x, w, ws), t3.linear_fp8(x[:3], w, ws)
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    assert t3.lib().t3_selftest_fp8_wait_runs_out(torch.cuda.current_stream().cuda_stream) == 0
    end.record()
    assert t3.device_error() == 4  # the first wait's bit alone: the second sees that the CTA has given up
    assert 0.5e3 < start.elapsed_time(end) < 10e3  # milliseconds: bounded, and not by a wait each
    assert t3.device_error() == 0
    assert torch.equal(t3.linear_fp8(x, w, ws), want[0]) and torch.equal(t3.linear_fp8(x[:3], w, ws), want[1])
