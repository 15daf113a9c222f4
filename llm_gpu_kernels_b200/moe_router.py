"""Routing to experts beyond softmax and top-k: score function, balance bias, expert groups, scaled weights.

The reference has one router, a formula in a capture script (scripts/capture_qwen3_moe_layer0.py:583-587: softmax over
all experts, top-k, divide by the sum of the k); that is the default ``RouterConfig()`` and what ``router_weight=`` of
the prepare functions runs without a ``router=``. Here the formula is a value:

    scores   s_e = softmax over the E logits of a token, or 1 / (1 + exp(-l_e))
    choice   c_e = s_e + bias_e; without a bias by the logits, which order the experts as the scores do
    groups   E / groups consecutive experts each, worth their largest c ("max") or the sum of their two largest
             ("top2"; of the scores without a bias); only the ``kept_groups`` best groups take part
    ids      the topk experts of largest c, in that order; ties, here and among groups, go to the lower index
    weights  the scores of those experts, divided by their sum if ``renormalize``, times ``scale``

An expert whose logit (or bias) is NaN or -inf is masked: it has no score and is never chosen while another is left;
slots that nobody can fill get the lowest unused indices with weight 0, so ids stay valid for the layer. Mask with -inf
(or the type's lowest value, which keeps an expert as a last resort): a mask like -1e9 leaves FP32 no room between the
other experts, and every row is routed in FP64, several times as long.

``prepare_routing`` routes logits a program already has; ``router=`` / ``router_bias=`` of ``prepare_moe`` and its
siblings configure the router that computes them from ``router_weight``. ``run()`` of either only enqueues kernels on
the current stream, so both can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import Optional

import torch

from . import _native, _ops

SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "top2": 1}
LOGIT_TYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.FP16, torch.float32: _native.FP32}


@dataclass(frozen=True)
class RouterConfig:
    """How logits become ids and weights; see the module's text for each field."""
    score: str = "softmax"
    groups: int = 1
    kept_groups: Optional[int] = None   # None: all of them
    group_score: str = "max"
    renormalize: bool = True
    scale: float = 1.0

    def __post_init__(self):
        if self.score not in SCORES:
            raise ValueError(f"unknown score {self.score!r}; expected one of {'/'.join(SCORES)}")
        if self.group_score not in GROUP_SCORES:
            raise ValueError(f"unknown group_score {self.group_score!r}; expected one of {'/'.join(GROUP_SCORES)}")
        if not 1 <= self.groups <= 32 or not 1 <= self.kept <= self.groups:
            raise ValueError("groups must be in [1,32] and kept_groups in [1,groups]")
        if not 0.0 < self.scale < float("inf"):
            raise ValueError("scale must be positive and finite")

    @property
    def kept(self):
        return self.groups if self.kept_groups is None else self.kept_groups

    def native(self):
        return _native.RouterConfig(score=SCORES[self.score], groups=self.groups, kept_groups=self.kept,
                                    group_score=GROUP_SCORES[self.group_score], renormalize=int(self.renormalize),
                                    scale=self.scale)

    def check(self, experts, topk):
        """Raises when ``topk`` experts cannot be chosen from ``experts`` in this way."""
        if experts % self.groups:
            raise ValueError(f"groups={self.groups} does not divide the {experts} experts")
        if not 1 <= topk <= min(32, self.kept * (experts // self.groups)):
            raise ValueError("router needs 1 <= topk <= 32 and topk <= experts of the kept groups")


def check_bias(bias, experts, device):
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.dtype != torch.float32
                             or tuple(bias.shape) != (experts,) or bias.device != device or not bias.is_contiguous()):
        raise ValueError("router bias must be a contiguous FP32 tensor [E] on the same device")


@dataclass
class PreparedRouting:
    """Fixed buffers; logits and bias may change in place between runs. ``ids`` and ``routing_weights`` are written by
    every ``run()`` and can be the tensors a prepared layer was given as its routes. No workspace: two prepared
    routings may run at the same time, one with itself may not."""
    logits: torch.Tensor
    topk: int
    config: RouterConfig
    bias: Optional[torch.Tensor]
    ids: torch.Tensor
    routing_weights: torch.Tensor
    _args: object = field(default=None, repr=False)
    _call: object = field(default=None, repr=False)
    _device: int = field(default=0, repr=False)
    _written: tuple = field(default=(), repr=False)

    def run(self):
        """Routes every row on the current stream; returns (ids, routing_weights)."""
        if _native.tracing():
            c = self.config
            _ops.route(self.logits, self.bias, self.ids, self.routing_weights, SCORES[c.score], c.groups, c.kept,
                       GROUP_SCORES[c.group_score], c.renormalize, float(c.scale))
        elif self.logits.shape[0]:
            _native.launch(self._call, self._args, self._device, self._written)
        return self.ids, self.routing_weights


def prepare_routing(logits, topk, *, config=RouterConfig(), bias=None, ids=None, routing_weights=None,
                    id_dtype=torch.int32):
    """Routing of ``logits`` [T,E] (BF16, FP16 or FP32; rows may be strided) to ``topk`` experts each. The outputs are
    allocated unless given: ``ids`` [T,topk] int32 / int64 and ``routing_weights`` [T,topk] FP32. Runs once."""
    if (not isinstance(logits, torch.Tensor) or logits.ndim != 2 or logits.dtype not in LOGIT_TYPES or not logits.is_cuda
            or (logits.shape[1] > 1 and logits.stride(1) != 1)
            or (logits.shape[0] > 1 and logits.stride(0) < logits.shape[1])):
        raise ValueError("expected CUDA BF16/FP16/FP32 logits [T,E] with contiguous rows that do not overlap")
    tokens, experts = logits.shape
    if not 0 < experts <= 256:
        raise ValueError("routing requires E in [1,256]")
    if not isinstance(config, RouterConfig):
        raise TypeError("config must be RouterConfig")
    topk = int(topk)
    config.check(experts, topk)
    if tokens * topk >= 2**31:
        raise ValueError("routing requires T*topk < 2**31")
    check_bias(bias, experts, logits.device)
    device = logits.device
    if ids is None:
        if id_dtype not in (torch.int32, torch.int64):
            raise ValueError("id_dtype must be torch.int32 or torch.int64")
        ids = torch.empty((tokens, topk), dtype=id_dtype, device=device)
    if routing_weights is None:
        routing_weights = torch.empty((tokens, topk), dtype=torch.float32, device=device)
    if (ids.dtype not in (torch.int32, torch.int64) or routing_weights.dtype != torch.float32
            or any(tuple(t.shape) != (tokens, topk) or t.device != device or not t.is_contiguous()
                   for t in (ids, routing_weights))):
        raise ValueError("expected contiguous CUDA IDs[T,topk] and FP32 weights of identical shape")
    _native.check_disjoint(written=(ids, routing_weights), read=(logits, bias))
    args = _native.RouteArgs(
        tokens=tokens, experts=experts, topk=topk, dtype=LOGIT_TYPES[logits.dtype],
        ids_are_int64=int(ids.dtype == torch.int64), pitch=logits.stride(0) if tokens > 1 else experts,
        config=config.native(), logits=logits.data_ptr(), bias=bias.data_ptr() if bias is not None else None,
        ids=ids.data_ptr(), weights=routing_weights.data_ptr())
    prepared = PreparedRouting(logits, topk, config, bias, ids, routing_weights, args, _native.load().b200moe_route,
                               device.index, (ids, routing_weights))
    prepared.run()
    return prepared
