"""The layer with experts in 8-bit integers (no counterpart in the reference, whose quantised experts are W4A16,
moe_w4_cuda.py:85-164).

    q(x)            rows of x as int8, one scale each (``int8_weights``)
    gate, up        = (q(x) . Wg^T, q(x) . Wu^T) * row scale * channel scale, integer sums
    a               = silu(gate) * up in FP32, quantised again row by row
    output          = sum over a token's routes of routing weight * (q(a) . Wd^T) * row scale * channel scale

Half the weight bytes of BF16 experts and twice their tensor rate. Life cycle, dispatch, combine, router and
attributes are those of ``prepare_moe``; ``activated`` and ``down_output`` are FP32 here, so that BF16 comes with the
result only, and ``x_q`` / ``x_scale`` / ``activated_q`` / ``activated_scale`` are the quantised rows, in grouped order. Any
H and I up to 131072 work (rows are padded to 16 bytes).
A token whose row holds an infinity or a NaN gives NaN in that row only.
"""
from .int8_weights import Int8Weight
from .moe import _prepare
from .moe_ranked import _ranked


def prepare_int8_moe(x, gate_up, down, ids, routing_weights, *, router_weight=None, router=None, router_bias=None,
                     router_bf16_weights=False, residual=None, token_tile=0):
    """``gate_up`` is an ``Int8Weight`` [E,2I,H] (gate rows, then up rows), ``down`` one [E,H,I]; the rest is as in
    ``prepare_moe``: x [T,H] BF16, ids and FP32 weights [T,K] (inputs, or with ``router_weight`` outputs)."""
    for weight, what in ((gate_up, "gate_up"), (down, "down")):
        if not isinstance(weight, Int8Weight):
            raise TypeError(f"{what} must be Int8Weight")
        if weight.values.ndim != 3 or not weight.values.is_cuda:
            raise ValueError(f"{what}: an Int8Weight [E,N,K] on a CUDA device required")
    return _ranked(_prepare(x, gate_up, down, ids, routing_weights, router_weight=router_weight, schedule="tcgen05",
                            token_tile=token_tile, router_bf16_weights=router_bf16_weights, residual=residual,
                            router=router, router_bias=router_bias))
