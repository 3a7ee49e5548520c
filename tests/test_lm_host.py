"""The feed-forward operators without a GPU: definitions, tasks, knobs, and what the C entries refuse before any launch."""
import ctypes

import pytest

from flextensor_b200 import backend
from flextensor_b200.ir import placeholder
from flextensor_b200.nn import ops
from flextensor_b200.scheduler import flatten_graph, schedule_with_config, schedule_with_config_ops
from flextensor_b200.space import generate_space_intra_op, op_family
from flextensor_b200.task import TASK_TABLE
from flextensor_b200.templates import config_to_knobs, knobs_to_config
from flextensor_b200.utils import Config

BAD_ARG, UNSUPPORTED, BAD_CONFIG, WORKSPACE, NO_DEVICE, TOO_LARGE = -1, -2, -3, -4, -6, -7


def bf(*shape):
    return placeholder(shape, dtype="bfloat16")


def test_linear_definition():
    out = ops.linear(bf(5, 64), bf(96, 64), bias=bf(96), residual=bf(5, 96), activation="gelu")
    assert tuple(int(s) for s in out.shape) == (5, 96) and out.dtype == "bfloat16"
    assert out.op.attrs["operands"] == ("x", "weight", "bias", "residual")
    assert [a.dom.extent.value for a in out.op.reduce_axis] == [64]
    gated = ops.linear(bf(5, 64), bf(96, 64), activation="silu", gated=True)
    assert tuple(int(s) for s in gated.shape) == (5, 48)
    for bad in (lambda: ops.linear(bf(5, 64), bf(96, 32)), lambda: ops.linear(bf(5, 64), bf(95, 64), gated=True),
                lambda: ops.linear(bf(5, 64), bf(96, 64), activation="tanh"),
                lambda: ops.linear(bf(5, 64), bf(96, 64), bias=bf(95)),
                lambda: ops.linear(placeholder((5, 64)), placeholder((96, 64))),
                lambda: ops.linear(bf(5, 64), bf(96, 64), residual=bf(4, 96))):
        with pytest.raises(AssertionError):
            bad()


def test_expert_definitions():
    ids, weights = ops.route_experts(placeholder((10, 8)), 2, scoring="sigmoid", groups=4, top_groups=2)
    assert ids.dtype == "int32" and weights.dtype == "float32" and ids.op is weights.op and ids.op.num_outputs == 2
    plan = ops.expert_plan(ids, 8)
    assert [tuple(int(s) for s in t.shape) for t in plan] == [(9,), (20,), (20,)]
    h = ops.expert_linear(bf(10, 64), bf(8, 96, 64), plan, gated=True, gather=True)
    assert tuple(int(s) for s in h.shape) == (20, 48)
    y = ops.expert_linear(h, bf(8, 64, 48), plan, bias=bf(8, 64))
    out = ops.expert_combine(y, plan, weights=weights, residual=bf(10, 64))
    assert tuple(int(s) for s in out.shape) == (10, 64)
    for bad in (lambda: ops.route_experts(placeholder((10, 8)), 9), lambda: ops.route_experts(placeholder((10, 8)), 2, groups=3),
                lambda: ops.route_experts(placeholder((10, 8)), 3, groups=4, top_groups=1),
                lambda: ops.expert_linear(bf(10, 64), bf(8, 96, 64), plan),          # sorted rows: 20 of them
                lambda: ops.expert_linear(bf(10, 64), bf(7, 96, 64), plan, gather=True),
                lambda: ops.expert_combine(bf(19, 64), plan), lambda: ops.expert_linear(h, bf(8, 64, 48), (ids, ids, ids))):
        with pytest.raises(AssertionError):
            bad()


def test_definitions_refuse_what_the_launchers_do():
    """Types, shapes and limits are named when the graph is made, not at its first run."""
    f32 = lambda *shape: placeholder(shape)
    i32 = lambda *shape: placeholder(shape, dtype="int32")
    plan = ops.expert_plan(i32(10, 2), 8)
    y, other = bf(20, 64), ops.expert_plan(i32(10, 2), 8)
    for bad in (lambda: ops.route_experts(placeholder((10, 8), dtype="int8"), 2), lambda: ops.route_experts(f32(2, 10, 8), 2),
                lambda: ops.route_experts(f32(10, 1025), 2), lambda: ops.route_experts(f32(10, 64), 33),
                lambda: ops.route_experts(f32(10, 66), 2, groups=33, top_groups=2),
                lambda: ops.route_experts(f32(10, 8), 2, bias=f32(7)), lambda: ops.route_experts(f32(10, 8), 2, bias=bf(8)),
                lambda: ops.expert_plan(i32(10, 2), 1025), lambda: ops.expert_plan(i32(10, 2), 0),
                lambda: ops.expert_plan(i32(10, 33), 64), lambda: ops.expert_plan(f32(10, 2), 8), lambda: ops.expert_plan(i32(20), 8),
                lambda: ops.expert_combine(f32(20, 64), plan), lambda: ops.expert_combine(y, plan, weights=f32(10, 3)),
                lambda: ops.expert_combine(y, plan, weights=bf(10, 2)), lambda: ops.expert_combine(y, plan, residual=f32(10, 64)),
                lambda: ops.expert_combine(y, plan, residual=bf(9, 64)),
                lambda: ops.expert_combine(y, (plan[0], plan[2], plan[1])), lambda: ops.expert_combine(y, (plan[0], plan[1], other[2]))):
        with pytest.raises(AssertionError):
            bad()
    for dtype in ("float32", "bfloat16", "float16"):
        ops.route_experts(placeholder((10, 1024), dtype=dtype), 32, bias=f32(1024), groups=32, top_groups=32)
    assert ops.expert_combine(y, plan, weights=f32(10, 2), residual=bf(10, 64)).dtype == "bfloat16"


def test_graph_order_and_plan():
    """Every op comes after its producers, though the router is reached over paths of three lengths."""
    key = "experts_expert_ffn_(8, 64, 8, 2048, 1024)_cuda(0)"
    task = TASK_TABLE[key]
    outs, bufs = task.func(*task.args)
    order, _ = flatten_graph(outs)
    assert [op.kind for op in order] == ["route_experts", "expert_plan", "expert_linear", "expert_linear", "expert_combine"]
    plan, bufs = schedule_with_config(key, Config([], None))
    assert [step.op.kind for step in plan.steps] == [op.kind for op in order] and len(bufs) == 12


def test_chain_order_is_unchanged():
    x, w, b = placeholder((2, 8, 10, 10)), placeholder((12, 8, 3, 3)), placeholder((12,))
    out = ops.relu(ops.conv2d_nchw(x, w, b, padding=1))
    assert [op.kind for op in flatten_graph([out.op])[0]] == ["pad2d", "conv2d", "bias_add", "relu"]


def test_knob_space_round_trip():
    out = ops.linear(bf(48, 512), bf(256, 512))
    assert op_family(out.op) == "linear"
    space = generate_space_intra_op(out.op, {})
    assert len(space) == 6 * 3 * 4 * 5
    knobs = {"tile_n": 64, "cluster": 1, "stages": 3, "split_k": 4}
    assert config_to_knobs(knobs_to_config(knobs, out.op), out.op) == knobs
    plan, _ = schedule_with_config_ops([out.op], list(out.op.input_tensors) + [out], Config([knobs_to_config(knobs, out.op)], None))
    assert plan.steps[0].knobs == knobs
    ids, _ = ops.route_experts(placeholder((10, 8)), 2)
    assert not generate_space_intra_op(ids.op, {}).subspaces


def test_every_linear_task_plans():
    keys = [k for k in TASK_TABLE if k.startswith(("linear_", "experts_")) and k.endswith("cuda(0)")]
    assert len(keys) >= 6
    for key in keys:
        schedule_with_config(key, Config([], None))


@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(1 << 16)
    base = ctypes.addressof(buf)
    yield ctypes.c_void_p((base + 255) // 256 * 256)
    del buf


def test_c_entries_refuse(native_lib, p):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    L = native_lib
    lin = lambda dtype=1, x=p, t=4, n=8, k=8, act=0, gated=0, cfg=None: L.ftb_linear(dtype, x, p, None, None, p, None, t, n, k, act, gated, cfg, None, None)
    assert lin() == NO_DEVICE
    assert lin(dtype=0) == BAD_ARG and lin(act=5) == BAD_ARG and lin(gated=2) == BAD_ARG and lin(x=None) == BAD_ARG
    assert lin(t=-1) == BAD_ARG and lin(n=0) == BAD_ARG and lin(k=0) == BAD_ARG
    assert lin(t=1 << 31) == TOO_LARGE
    assert lin(t=0, x=None) == 0                                  # nothing to do
    for knobs in ({"tile_n": 24}, {"tile_n": 512}, {"cluster": 3}, {"split_k": 3}, {"split_k": 2, "cluster": 2},
                  {"split_k": 2, "tile_n": 128}, {"stages": 9}, {"tile_n": 256, "cluster": 1}, {"tile_n": 64, "cluster": 2}):
        assert lin(cfg=ctypes.byref(backend.FtbConfig.from_dict(knobs))) == BAD_CONFIG, knobs
    need = backend.linear_backward_workspace_bytes(4, 8, 8, True)
    back = lambda ws=p, size=need, dx=p, z=p, gated=1, dw=None: L.ftb_linear_backward(1, p, p, p, z, dx, dw, None, 4, 8, 8, 0, gated, ws, size, None, None)
    assert back() == NO_DEVICE and back(dx=None) == BAD_ARG and back(z=None) == BAD_ARG
    assert back(size=need - 1) == WORKSPACE and back(ws=None) == WORKSPACE
    assert back(ws=ctypes.c_void_p(p.value + 8)) == WORKSPACE
    route = lambda dtype=0, t=4, e=8, k=2, scoring=0, g=1, tg=1, logits=p: L.ftb_route_experts(dtype, logits, None, p, p, t, e, k, scoring, g, tg, 1, 1.0, None)
    assert route() == NO_DEVICE and route(t=0, logits=None) == 0
    assert route(dtype=3) == BAD_ARG and route(k=9) == BAD_ARG and route(g=3) == BAD_ARG and route(tg=2) == BAD_ARG
    assert route(scoring=2) == BAD_ARG and route(g=4, tg=1, k=3) == BAD_ARG and route(logits=None) == BAD_ARG
    assert route(e=1025) == TOO_LARGE and route(e=64, k=33) == TOO_LARGE and route(e=64, g=64, tg=2, k=1) == TOO_LARGE
    plan = lambda rows=4, e=8, ids=p: L.ftb_expert_plan(ids, p, p, p, rows, e, None)
    assert plan() == NO_DEVICE and plan(rows=-1) == BAD_ARG and plan(e=0) == BAD_ARG and plan(ids=None) == BAD_ARG
    assert plan(e=1025) == TOO_LARGE
    el = lambda rows=4, k=2, e=8, gather=0, order=p, cfg=None: L.ftb_expert_linear(1, p, p, None, p, order, p, None, rows, k, e, 8, 8, 0, 0, gather, cfg, None, None)
    assert el() == NO_DEVICE and el(rows=5) == BAD_ARG and el(gather=2) == BAD_ARG and el(gather=1, order=None) == BAD_ARG
    assert el(k=33, rows=66) == TOO_LARGE and el(rows=0) == 0
    assert el(cfg=ctypes.byref(backend.FtbConfig.from_dict({"split_k": 2}))) == BAD_CONFIG
    combine = lambda t=4, k=2, y=p: L.ftb_expert_combine(1, y, p, None, None, p, t, k, 8, None)
    assert combine() == NO_DEVICE and combine(y=None) == BAD_ARG and combine(t=-1) == BAD_ARG and combine(t=0, y=None) == 0
    cb = lambda dy=p, dw=None, y=None: L.ftb_expert_combine_backward(1, p, y, p, None, dy, dw, 4, 2, 8, None)
    assert cb() == NO_DEVICE and cb(dy=None) == BAD_ARG and cb(dw=p) == BAD_ARG
    assert L.ftb_launch_count() == 0


def test_python_refuses_cpu_tensors():
    import torch
    x, w, out = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        backend.linear(x, w, out)
    with pytest.raises(TypeError):
        backend.route_experts(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2))
    with pytest.raises(ValueError):
        backend.ExpertPlan(4, 33, 64, device="cpu")
    with pytest.raises(TypeError):
        backend.expert_plan(torch.zeros(4, 2, dtype=torch.int32), backend.ExpertPlan(4, 2, 8, device="cpu"))
