"""One dense product in 8-bit integers: y = (q(x) . W^T) * row scale * channel scale.

    scale[t] = max_k |x[t,k]| / 127    q[t,k] = rint(127 x[t,k] / max_k |x[t,k]|), ties to even
    y[t,n] = (sum_k q[t,k] W[n,k]) * scale[t] * w_scale[n]

The sums are exact integers; y is rounded once, to the type of x. A row that holds an infinity or a NaN gives NaN. The
same kernels run the experts of ``moe_int8_cuda``; this is the projection without experts (a shared expert, a gate,
an output projection next to the layer). Prepared like the layer: fixed buffers and shapes, values change in place,
``run()`` only enqueues kernels on the current stream and can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import torch

from . import _native, _ops
from .int8_weights import Int8Weight

_TYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.FP16}


@dataclass
class PreparedInt8Linear:
    """One workspace: never run concurrently with itself; the caller orders streams."""
    x: torch.Tensor
    weight: Int8Weight
    output: torch.Tensor
    x_q: torch.Tensor        # [T, K rounded up to 16] int8, rewritten by every run
    x_scale: torch.Tensor    # [T] FP32
    status: torch.Tensor
    kernel_launches: int = 0
    _plan: object = field(default=None, repr=False)
    _call: object = field(default=None, repr=False)
    _device: int = field(default=0, repr=False)
    _written: tuple = field(default=(), repr=False)

    def run(self):
        """One product on the current stream; returns ``output``."""
        if _native.tracing():
            _ops.int8_linear(self._plan.value, self.x, self.weight.storage, self.weight.scales, self.output, self.x_q,
                             self.x_scale, self.status)
        elif self.x.shape[0]:
            _native.launch(self._call, self._plan, self._device, self._written)
        return self.output

    def check(self):
        """Explicit synchronising check of the status word."""
        flags = int(self.status.item())
        if flags:
            raise RuntimeError(f"int8 product: GPU status={flags} (4=kernel wait timeout)")

    def __del__(self):
        plan, self._plan = self._plan, None
        if plan is not None:
            try:
                _native.load().b200moe_linear_destroy(plan)
            except Exception:  # interpreter shutdown
                pass


def prepare_int8_linear(x, weight, *, output=None):
    """Product of ``x`` [T,K] (BF16 or FP16, rows may be strided) with an ``Int8Weight`` [N,K]; ``output`` [T,N] of the
    type of x is allocated unless given. Runs once."""
    if (not isinstance(x, torch.Tensor) or x.ndim != 2 or x.dtype not in _TYPES or not x.is_cuda
            or (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1])):
        raise ValueError("expected a CUDA BF16/FP16 tensor [T,K] with contiguous rows that do not overlap")
    if not isinstance(weight, Int8Weight):
        raise TypeError("weight must be Int8Weight")
    if weight.values.ndim != 2 or weight.shape[1] != x.shape[1] or weight.device != x.device:
        raise ValueError("weight must be an Int8Weight [N,K] on the device of x")
    tokens, k = x.shape
    n = weight.shape[0]
    device = x.device
    if output is None:
        output = torch.empty((tokens, n), dtype=x.dtype, device=device)
    elif (not isinstance(output, torch.Tensor) or tuple(output.shape) != (tokens, n) or output.dtype != x.dtype
          or output.device != device or not output.is_contiguous()):
        raise ValueError("output must be a contiguous tensor [T,N] of the type and device of x")
    _native.check_disjoint(written=(output,), read=(x, weight.storage, weight.scales))
    lib = _native.load()
    shape = _native.LinearShape(tokens=tokens, k=k, n=n, dtype=_TYPES[x.dtype])
    handle = ctypes.c_void_p()
    _native.check(lib.b200moe_linear_create(ctypes.byref(shape), ctypes.byref(handle)))
    try:
        sizes = _native.LinearWorkspace()
        _native.check(lib.b200moe_linear_workspace(handle, ctypes.byref(sizes)))
        prepared = PreparedInt8Linear(
            x, weight, output, torch.empty((tokens, sizes.x_q // max(1, tokens)), dtype=torch.int8, device=device),
            torch.empty((tokens,), dtype=torch.float32, device=device),
            torch.zeros((1,), dtype=torch.int32, device=device), kernel_launches=sizes.launches)
        ptr = lambda t: t.data_ptr() if t.numel() else None
        buffers = _native.LinearBuffers(
            x=ptr(x), x_pitch=x.stride(0) if tokens > 1 else k, weight=ptr(weight.storage), weight_scale=ptr(weight.scales),
            output=ptr(output), x_q=ptr(prepared.x_q), x_scale=ptr(prepared.x_scale), status=ptr(prepared.status))
        with torch.cuda.device(device):
            _native.check(lib.b200moe_linear_bind(handle, ctypes.byref(buffers)))
    except Exception:
        lib.b200moe_linear_destroy(handle)
        raise
    prepared._plan, prepared._call, prepared._device = handle, lib.b200moe_linear_forward, device.index
    prepared._written = (output, prepared.x_q, prepared.x_scale, prepared.status)
    _ops.register_linear(prepared)
    prepared.run()
    return prepared
