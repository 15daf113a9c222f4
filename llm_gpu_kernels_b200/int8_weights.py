"""Weights in 8-bit integers with one FP32 scale per output channel.

    scale[n] = max_k |w[n,k]| / 127        value[n,k] = rint(w[n,k] / scale[n]) in [-127, 127]

The activations of a product with such a weight are quantised the same way, one scale per row, by the kernel that runs
it (``int8_linear``, ``moe_int8_cuda``). The reference has no integer format with per-channel scales; its packed int4
format (moe_weight_quant.py) keeps BF16 activations.
"""
from __future__ import annotations

import torch

MAX_K = 131072   # inputs of one product: its sums must fit 32 bits


def row_pitch(k: int) -> int:
    """Bytes from one weight row to the next in the layout the kernels read."""
    return (k + 15) // 16 * 16


class Int8Weight:
    """``values`` int8 [N,K] or [E,N,K] and ``scales`` FP32 [N] or [E,N], immutable. ``storage`` is the layout the kernels
    read: the values themselves where K is a multiple of 16 and they are contiguous and 16-byte aligned, else a copy
    with rows padded to a multiple of 16 bytes, made here once."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if (not isinstance(values, torch.Tensor) or not isinstance(scales, torch.Tensor) or values.dtype != torch.int8
                or scales.dtype != torch.float32 or values.ndim not in (2, 3) or scales.shape != values.shape[:-1]
                or values.device != scales.device or not scales.is_contiguous() or 0 in values.shape):
            raise ValueError("int8 weight: int8 values [N,K] or [E,N,K] and contiguous FP32 scales [N] or [E,N] required")
        if values.shape[-1] > MAX_K:
            raise ValueError(f"int8 weight: K is at most {MAX_K} (32-bit sums)")
        self.values = values
        self.scales = scales
        k = values.shape[-1]
        if k % 16 == 0 and values.is_contiguous() and values.data_ptr() % 16 == 0:
            self.storage = values
        else:
            self.storage = torch.zeros(*values.shape[:-1], row_pitch(k), dtype=torch.int8, device=values.device)
            self.storage[..., :k] = values

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    def to(self, device):
        return Int8Weight(self.values.to(device), self.scales.to(device))

    def dequantize(self):
        """FP32 values the weight stands for."""
        return self.values.float() * self.scales[..., None]


def quantize_int8(weight: torch.Tensor) -> Int8Weight:
    """Quantise a BF16 / FP16 / FP32 weight [N,K] or [E,N,K] channel by channel, on the device it is on."""
    if (not isinstance(weight, torch.Tensor) or weight.ndim not in (2, 3) or 0 in weight.shape
            or weight.dtype not in (torch.bfloat16, torch.float16, torch.float32)):
        raise ValueError("expected a BF16/FP16/FP32 weight [N,K] or [E,N,K]")
    parts = weight if weight.ndim == 3 else weight[None]
    values = torch.empty(parts.shape, dtype=torch.int8, device=weight.device)
    scales = torch.empty(parts.shape[:-1], dtype=torch.float32, device=weight.device)
    for e in range(parts.shape[0]):   # one expert at a time bounds the FP32 temporaries
        w = parts[e].float()
        top = w.abs().amax(-1, keepdim=True)
        if not bool(torch.isfinite(top).all()):
            raise ValueError("weight holds an infinity or a NaN")
        scales[e] = top[:, 0] / 127
        # 127 w in FP64: exact for tiny and huge rows alike
        values[e] = torch.where(top > 0, torch.round(127 * w.double() / top.double().clamp_min(1e-300)), 0.0).to(torch.int8)
    return Int8Weight(values if weight.ndim == 3 else values[0], scales if weight.ndim == 3 else scales[0])
