"""CPU-only checks of the 8-bit layers' and the router's entry points: every refusal by its name, before the device is touched, and the
workspaces' sizes."""
import ctypes as C

import pytest
import torch

import turboexl3_b200 as t3
from turboexl3_b200 import api

FAKE = 0x1000  # non-null and 256-byte aligned; a refusal never dereferences it


def name(status):
    return t3.status_name(status)


def _route(logits=FAKE, dtype=0, rows=1, experts=64, topk=4, scoring=0, bias=None, groups=1, group_topk=1, scale=1.0, inds=FAKE, scores=FAKE):
    return name(t3.lib().t3_route(logits, dtype, rows, experts, topk, scoring, bias, groups, group_topk, 1, scale, inds, scores, None))


def test_route_refusals():
    assert _route(logits=None) == "NullPointer"
    assert _route(inds=None) == "NullPointer"
    assert _route(scores=None) == "NullPointer"
    assert _route(dtype=3) == "BadExl3Dtype"
    assert _route(scoring=2) == "Exl3EngineNotImplemented"
    for bad in (dict(rows=0), dict(experts=0), dict(experts=1025), dict(topk=0), dict(topk=33), dict(experts=3, topk=4), dict(groups=0),
                dict(groups=33, experts=66), dict(groups=5), dict(groups=8, group_topk=9), dict(groups=8, group_topk=0),
                dict(groups=32, group_topk=1, topk=3), dict(group_topk=2), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert _route(**bad) == "BadExl3Shape", bad


def _quantize(x=FAKE, dt=2, rows=1, width=256, q=FAKE, scale=FAKE):
    return name(t3.lib().t3_quantize_fp8(x, dt, rows, width, q, scale, None))


def test_quantize_refusals():
    for bad in (dict(x=None), dict(q=None), dict(scale=None)):
        assert _quantize(**bad) == "NullPointer"
    assert _quantize(dt=3) == "BadExl3Dtype"
    for bad in (dict(rows=0), dict(width=0), dict(width=200), dict(width=-128), dict(x=FAKE + 8), dict(q=FAKE + 8)):
        assert _quantize(**bad) == "BadExl3Shape", bad


def _linear(x=FAKE, dt=2, xs=None, rows=1, w=FAKE, ws=FAKE, width=256, out=256, y=FAKE, ydt=2, work=FAKE, work_bytes=1 << 40):
    return name(t3.lib().t3_linear_fp8(x, dt, xs, rows, w, ws, width, out, y, ydt, work, work_bytes, None))


def test_linear_refusals():
    for bad in (dict(x=None), dict(w=None), dict(ws=None), dict(y=None), dict(dt=3, xs=None)):
        assert _linear(**bad) == "NullPointer", bad
    for bad in (dict(dt=4), dict(dt=-1), dict(ydt=3)):
        assert _linear(**bad) == "BadExl3Dtype", bad
    for bad in (dict(rows=0), dict(width=0), dict(width=200), dict(out=0), dict(out=-1), dict(xs=FAKE), dict(x=FAKE + 4), dict(w=FAKE + 8),
                dict(y=FAKE + 2), dict(rows=1 << 23, width=1024)):
        assert _linear(**bad) == "BadExl3Shape", bad
    assert _linear(rows=200, work=None) == "NullPointer"
    assert _linear(rows=200, work_bytes=16) == "WorkspaceTooSmall"
    assert _linear(rows=200, work=FAKE + 16) == "WorkspaceTooSmall"


def test_linear_past_decode_rows_follows_the_configuration():
    t3.configure(prefill=False)
    try:
        assert _linear(rows=33) == "Exl3EngineNotImplemented"
    finally:
        t3.configure()


def test_linear_workspace():
    L = t3.lib()
    assert L.t3_linear_fp8_workspace_bytes(1, 2048, 2048, 2) == 0            # the kernel quantises the row itself
    assert L.t3_linear_fp8_workspace_bytes(200, 2048, 2048, api.E4M3) == 0   # quantised already
    assert L.t3_linear_fp8_workspace_bytes(200, 2048, 2048, 2) >= 200 * (2048 + 16 * 4)
    assert L.t3_linear_fp8_workspace_bytes(0, 2048, 2048, 2) == 0


def _bank(experts=8, hidden=256, inter=128, **null):
    p = [api._Fp8Proj(null.get("w", FAKE), null.get("scale", FAKE)) for _ in range(3)]
    return api._Fp8Bank(*p, experts, hidden, inter)


def _moe(bank=None, x=FAKE, dt=2, rows=1, inds=FAKE, scores=FAKE, sdt=0, topk=2, shared=None, y=FAKE, work=FAKE, work_bytes=1 << 40):
    b = bank or _bank()
    return name(t3.lib().t3_moe_fp8(x, dt, rows, C.byref(b), inds, scores, sdt, topk, shared, y, work, work_bytes, None))


def test_moe_refusals():
    for bad in (dict(x=None), dict(inds=None), dict(scores=None), dict(y=None), dict(work=None), dict(bank=_bank(w=None)),
                dict(bank=_bank(scale=None))):
        assert _moe(**bad) == "NullPointer", bad
    for bad in (dict(dt=3), dict(sdt=3)):
        assert _moe(**bad) == "BadExl3Dtype", bad
    for bad in (dict(bank=_bank(hidden=200)), dict(bank=_bank(inter=64)), dict(bank=_bank(experts=0)), dict(bank=_bank(experts=2049)),
                dict(bank=_bank(experts=2048, hidden=1 << 20)), dict(rows=0), dict(topk=0), dict(topk=33), dict(x=FAKE + 8), dict(y=FAKE + 8), dict(shared=FAKE + 8),
                dict(bank=_bank(w=FAKE + 8))):
        assert _moe(**bad) == "BadExl3Shape", bad
    assert _moe(rows=33) == "Exl3EngineNotImplemented"
    assert _moe(work_bytes=16) == "WorkspaceTooSmall"
    assert _moe(work=FAKE + 16) == "WorkspaceTooSmall"


@pytest.mark.parametrize("rows,topk,experts,hidden,inter", [(1, 1, 1, 128, 128), (32, 32, 2048, 7168, 2048), (32, 10, 512, 2048, 512), (17, 8, 64, 16384, 4096)])
def test_moe_workspace_covers_the_experts_in_use(rows, topk, experts, hidden, inter):
    b = _bank(experts, hidden, inter)
    used, cap = min(experts, rows * topk), 16 if rows <= 16 else 32
    assert t3.lib().t3_moe_fp8_workspace_bytes(rows, topk, C.byref(b)) >= used * cap * (inter + inter // 128 * 4)


def test_python_refusals():
    x, logits = torch.zeros(2, 256), torch.zeros(2, 64)
    w, s = torch.zeros(256, 256).to(torch.float8_e4m3fn), torch.ones(2, 2)
    for call in (lambda: t3.route(logits, 4), lambda: t3.quantize_fp8(x), lambda: t3.linear_fp8(x, w, s)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(t3.Exl3Error, match="Exl3EngineNotImplemented"):
        t3.route(logits, 4, "tanh")
    with pytest.raises(t3.Exl3Error, match="BadExl3Dtype"):
        t3.linear_fp8(x, w, s, out_dtype=torch.int8)


@pytest.mark.parametrize("rows", [1, 2, 16, 17, 32])
@pytest.mark.parametrize("width", [128, 1024, 7168, 16384, 131072, 1 << 20])
def test_every_width_has_a_plan(rows, width):
    """Where rows are quantised ahead, a call with a byte too little gets past the plan and is refused for the workspace."""
    L = t3.lib()
    for out in (1, 128, 576, 1000):
        need = L.t3_linear_fp8_workspace_bytes(rows, width, out, 2)
        if need:
            assert need >= rows * (width + width // 32)
            assert _linear(rows=rows, width=width, out=out, work_bytes=need - 1) == "WorkspaceTooSmall"


@pytest.mark.parametrize("hidden", [128, 1024, 7168, 32768])
@pytest.mark.parametrize("inter", [128, 2048, 16384])
def test_every_layer_has_a_plan(hidden, inter):
    L = t3.lib()
    for experts in (1, 8, 512, 2048):
        for rows in (1, 16, 17, 32):
            for topk in (1, 8, 32):
                if experts * max(hidden, inter) < 1 << 31:
                    b = _bank(experts, hidden, inter)
                    assert L.t3_moe_fp8_workspace_bytes(rows, topk, C.byref(b)) > 0


class _GemmPlan(C.Structure):
    _fields_ = [("n", C.c_uint32), ("split", C.c_uint32), ("grid", C.c_uint32)]


def _gemm_plan():
    plan = t3.lib()._ZN2t313plan_fp8_gemmEjjj  # t3::plan_fp8_gemm(rows, in, out)
    plan.restype, plan.argtypes = _GemmPlan, [C.c_uint32] * 3
    return plan


def test_the_shapes_tested_on_the_device_reach_every_kernel_of_the_gemm():
    from fp8_shapes import GEMM
    if torch.cuda.is_available() and torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the plans of 148 multiprocessors")
    plan = _gemm_plan()
    for shape, kernel in GEMM.items():
        p = plan(*shape)
        assert (p.n, p.split) == kernel, shape
    reached = set()
    for rows in list(range(33, 700, 13)) + [1000, 2000, 8192]:
        for width in list(range(128, 2048, 128)) + list(range(2048, 20481, 512)):
            for out in (64, 77, 200, 576, 700, 1100, 1601, 3001, 6144):
                p = plan(rows, width, out)
                assert p.n in (64, 128, 256) and 1 <= p.grid <= 148 and p.split <= 8 and p.grid % p.split == 0
                assert p.split == 1 or p.grid == -(-rows // 128) * -(-out // p.n) * p.split
                reached.add((p.n, p.split))
    assert reached == set(GEMM.values())


@pytest.mark.parametrize("rows,topk,served", [(1, 1, 79872), (16, 32, 79872), (17, 1, 34816), (32, 32, 34816)])
def test_hidden_sizes_of_the_routed_layer_that_are_served(rows, topk, served):
    """Every one up to what the header states; past some larger one none, by the same status from the call, and a workspace of 0."""
    L = t3.lib()

    def need(experts, hidden):
        return L.t3_moe_fp8_workspace_bytes(rows, topk, C.byref(_bank(experts, hidden, 128)))
    for experts in (1, 64, 2048):
        assert all(need(experts, h) > 0 for h in range(128, served + 1, 128))
        end = next(h for h in range(served, 200000, 128) if need(experts, h) == 0)
        assert all(need(experts, h) == 0 for h in range(end, end + 40000, 128))
        for h, status in ((end - 128, "WorkspaceTooSmall"), (end, "Exl3EngineNotImplemented")):
            assert _moe(bank=_bank(experts, h, 128), rows=rows, topk=topk, work_bytes=16) == status


def test_linear_rows_that_are_served():
    assert _linear(rows=65535 * 64, width=128, out=511, work_bytes=16) == "WorkspaceTooSmall"
    assert _linear(rows=65535 * 64, width=128, out=513, work_bytes=16) == "BadExl3Shape"
    assert _linear(rows=65535 * 64 + 1, width=128, out=1, work_bytes=16) == "BadExl3Shape"
