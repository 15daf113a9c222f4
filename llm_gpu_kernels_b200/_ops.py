"""``torch.library`` registration of the forward: ``torch.ops.b200moe.forward``.

The C ABI (``b200moe_forward``) takes raw pointers bound at prepare time, so the
operator proper is "enqueue the plan's kernels on the current stream". Wrapping
that call as a PyTorch custom op tells PyTorch which tensors it writes, which is
what lets ``PreparedMoE.run()`` sit inside ``torch.cuda.graph`` capture and inside
a ``torch.compile(fullgraph=True)`` region without a graph break: the tracer sees
one opaque op that mutates ``output`` (and the workspace, and ``ids`` /
``routing_weights`` when the plan has a router) and reads the rest.

The reference reaches its native plans through pybind11 classes holding
``torch::Tensor`` members (cuda_gate_up.cu:133-191); this is the same boundary with
the tensors passed per call for the tracer's benefit and the addresses fixed in the plan.
"""
from __future__ import annotations

import weakref
from typing import List, Optional

import torch

from . import _native

_LIB_NAME = "b200moe::forward"
_PLANS = {}   # plan address -> weak reference to the PreparedMoE that owns it


def register_plan(prepared):
    """Called by ``PreparedMoE.run()`` once: lets the operator find the tensors bound into the plan."""
    key = prepared._plan.value
    _PLANS[key] = weakref.ref(prepared, lambda _ref, key=key: _PLANS.pop(key, None))


def _bound_tensors(prepared):
    bound = [prepared.ids, prepared.routing_weights, prepared.output, prepared.counts, prepared.offsets,
             prepared.cursors, prepared.tasks, prepared.mapping, prepared.ranks, prepared.grouped_input,
             prepared.activated, prepared.down_output, prepared.status, prepared.scratch]
    if prepared.source_rows is not None:
        bound.append(prepared.source_rows)
    return bound + prepared.int8_workspace()


@torch.library.custom_op(_LIB_NAME, mutates_args=("ids", "routing_weights", "output", "workspace"),
                         device_types="cuda")
def forward(plan: int, x: torch.Tensor, weights: List[torch.Tensor], ids: torch.Tensor,
            routing_weights: torch.Tensor, output: torch.Tensor, workspace: List[torch.Tensor]) -> None:
    """One forward of the prepared plan ``plan`` (the ``B200MoePlan*`` as an integer) on the current stream of
    ``x``'s device. The kernels use the addresses bound at prepare time; the tensor arguments tell PyTorch what
    is read and what is written. Normally they ARE the bound tensors and nothing else happens. A tracer that
    functionalises the call (``torch.compile`` without re-inplacing) hands in copies instead: values of passed
    inputs are then copied into the bound buffers before the forward and the bound results into the passed
    tensors after it, so the op is a function of its arguments either way."""
    device = x.device
    lib = _native.load()
    owner = _PLANS.get(plan)
    prepared = owner() if owner is not None else None
    passed = [ids, routing_weights, output, *workspace]
    bound = _bound_tensors(prepared) if prepared is not None else passed
    if prepared is not None:
        for given, real in ((x, prepared.x), (ids, prepared.ids), (routing_weights, prepared.routing_weights),
                            *zip(weights, prepared._op_args[2])):
            if given.data_ptr() != real.data_ptr():
                real.copy_(given)
    if torch.cuda.current_device() == device.index:
        _native.check(lib.b200moe_forward(plan, torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            _native.check(lib.b200moe_forward(plan, torch.cuda.current_stream(device).cuda_stream))
    for given, real in zip(passed, bound):
        if given.data_ptr() != real.data_ptr():
            given.copy_(real)


@forward.register_fake
def _(plan, x, weights, ids, routing_weights, output, workspace):
    return None


@torch.library.custom_op("b200moe::route", mutates_args=("ids", "routing_weights"), device_types="cuda")
def route(logits: torch.Tensor, bias: Optional[torch.Tensor], ids: torch.Tensor, routing_weights: torch.Tensor,
          score: int, groups: int, kept_groups: int, group_score: int, renormalize: bool, scale: float) -> None:
    """Routing of given logits (``b200moe_route``) for tracers; ``PreparedRouting.run()`` calls it while compiling."""
    if logits.shape[0] == 0:
        return
    types = {torch.bfloat16: _native.BF16, torch.float16: _native.FP16, torch.float32: _native.FP32}
    rows = logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()
    args = _native.RouteArgs(
        tokens=rows.shape[0], experts=rows.shape[1], topk=ids.shape[1], dtype=types[rows.dtype],
        ids_are_int64=int(ids.dtype == torch.int64), pitch=rows.stride(0) if rows.shape[0] > 1 else rows.shape[1],
        config=_native.RouterConfig(score=score, groups=groups, kept_groups=kept_groups, group_score=group_score,
                                    renormalize=int(renormalize), scale=scale),
        logits=rows.data_ptr(), bias=bias.data_ptr() if bias is not None else None, ids=ids.data_ptr(),
        weights=routing_weights.data_ptr())
    _native.launch(_native.load().b200moe_route, args, rows.device.index, ())   # the operator declares what it writes


@route.register_fake
def _(logits, bias, ids, routing_weights, score, groups, kept_groups, group_score, renormalize, scale):
    return None


@torch.library.custom_op("b200moe::int8_linear", mutates_args=("output", "x_q", "x_scale", "status"), device_types="cuda")
def int8_linear(plan: int, x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, output: torch.Tensor,
                x_q: torch.Tensor, x_scale: torch.Tensor, status: torch.Tensor) -> None:
    """One product of the prepared plan (``b200moe_linear_forward``) for tracers. The kernels use the addresses bound at
    prepare time; where a tracer passes copies, values are copied in and out as for ``forward``."""
    owner = _LINEARS.get(plan)
    prepared = owner() if owner is not None else None
    if prepared is None:
        raise RuntimeError("int8 product: its prepared object is gone")
    if x.shape[0] == 0:
        return
    if x.data_ptr() != prepared.x.data_ptr():
        prepared.x.copy_(x)
    _native.launch(prepared._call, prepared._plan, prepared._device, ())
    for given, real in ((output, prepared.output), (x_q, prepared.x_q), (x_scale, prepared.x_scale),
                        (status, prepared.status)):
        if given.data_ptr() != real.data_ptr():
            given.copy_(real)


@int8_linear.register_fake
def _(plan, x, weight, weight_scale, output, x_q, x_scale, status):
    return None


_LINEARS = {}   # plan address -> weak reference to the PreparedInt8Linear that owns it


def register_linear(prepared):
    key = prepared._plan.value
    _LINEARS[key] = weakref.ref(prepared, lambda _ref, key=key: _LINEARS.pop(key, None))
