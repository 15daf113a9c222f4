"""ctypes binding of libb200moe.so (the C ABI declared in include/b200moe.h).

The library is the only compute path: if it is missing or does not export the
expected ABI this module raises; there is no fallback of any kind.
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch
from torch.overrides import _get_current_function_mode_stack
from torch.utils._device import DeviceContext

LIBRARY_PATH = Path(__file__).resolve().parent / "libb200moe.so"
ABI_VERSION = 6

STATUS_BAD_ID = 1
STATUS_BAD_WEIGHT = 2
STATUS_TIMEOUT = 4
STATUS_EP_OVERFLOW = 8

WEIGHTS_BF16 = 0
WEIGHTS_W4G128 = 1
WEIGHTS_INT8 = 2

BF16, FP16, FP32 = 0, 1, 2   # element types of operators that take more than BF16

SCHEDULE_AUTO = 0
SCHEDULE_GENERIC = 1
SCHEDULE_TCGEN05 = 2
SCHEDULE_NAMES = {SCHEDULE_GENERIC: "generic", SCHEDULE_TCGEN05: "tcgen05"}

ERR_INVALID, ERR_CUDA, ERR_UNSUPPORTED, ERR_STATE = -1, -2, -3, -4


class RouterConfig(ctypes.Structure):
    """``B200MoeRouterConfig``."""
    _fields_ = [(name, ctypes.c_int32) for name in (
        "score", "groups", "kept_groups", "group_score", "renormalize", "bf16_weights")] + [
        ("scale", ctypes.c_float), ("reserved", ctypes.c_int32)]


class Shape(ctypes.Structure):
    _fields_ = [(name, ctypes.c_int32) for name in (
        "tokens", "experts", "topk", "hidden", "intermediate", "ids_are_int64", "gate_up_format",
        "down_format", "schedule", "token_tile", "use_router", "route_only", "external_dispatch", "router_bf16_weights",
        "unchained", "fused_gather", "down_tiles")] + [("reserved", ctypes.c_int32 * 1), ("router", RouterConfig)]


WORKSPACE_BUFFERS = ("output", "counts", "offsets", "cursors", "tasks", "mapping", "ranks",
                     "grouped_input", "activated", "down_output", "status", "scratch")

INT8_BUFFERS = ("x_q", "x_scale", "activated_q", "activated_scale")


class Workspace(ctypes.Structure):
    _fields_ = [(name, ctypes.c_size_t) for name in WORKSPACE_BUFFERS + ("source_rows",) + INT8_BUFFERS] + [
        ("token_tile", ctypes.c_int32), ("schedule", ctypes.c_int32), ("launches", ctypes.c_int32),
        ("gathers", ctypes.c_int32), ("down_tiles", ctypes.c_int32), ("reserved", ctypes.c_int32)]


INPUT_BUFFERS = ("x", "router_weight", "gate_up", "gate_up_scales", "down", "down_scales", "ids",
                 "routing_weights")


class Buffers(ctypes.Structure):
    _fields_ = [(name, ctypes.c_void_p) for name in INPUT_BUFFERS + WORKSPACE_BUFFERS + (
        "valid_routes", "residual", "ep_row_dest", "ep_return_bases", "source_rows", "router_bias") + INT8_BUFFERS]


class RouteArgs(ctypes.Structure):
    """``B200MoeRouteArgs``: routing on given logits."""
    _fields_ = [(name, ctypes.c_int32) for name in (
        "tokens", "experts", "topk", "dtype", "ids_are_int64", "reserved")] + [
        ("pitch", ctypes.c_int64), ("config", RouterConfig)] + [
        (name, ctypes.c_void_p) for name in ("logits", "bias", "ids", "weights")]


class LinearShape(ctypes.Structure):
    """``B200MoeLinearShape``: one dense product in 8-bit integers."""
    _fields_ = [(name, ctypes.c_int32) for name in ("tokens", "k", "n", "dtype")] + [("reserved", ctypes.c_int32 * 4)]


class LinearWorkspace(ctypes.Structure):
    _fields_ = [(name, ctypes.c_size_t) for name in ("x_q", "x_scale", "status")] + [
        ("launches", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class LinearBuffers(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("x_pitch", ctypes.c_int64)] + [
        (name, ctypes.c_void_p) for name in ("weight", "weight_scale", "output", "x_q", "x_scale", "status")]


class DispatchArgs(ctypes.Structure):
    """Arguments of ``b200moe_dispatch_static`` (the entry point that allocates nothing)."""
    _fields_ = [(name, ctypes.c_int32) for name in (
        "tokens", "experts", "topk", "hidden", "ids_are_int64", "token_tile")] + [
        (name, ctypes.c_void_p) for name in (
            "x", "ids", "routing_weights", "counts", "offsets", "cursors", "tasks", "ranks", "mapping",
            "grouped_input", "status")]


STATIC_DISPATCH_MAX_ROUTES = 65536
EP_MAX_RANKS = 8


class EpArgs(ctypes.Structure):
    """``B200MoeEpArgs``: expert parallelism over peer memory."""
    _fields_ = [(name, ctypes.c_int32) for name in (
        "rank", "world", "experts", "topk", "hidden", "tokens", "capacity", "token_tile", "ids_are_int64",
        "fused_return")] + [("reserved", ctypes.c_int32 * 2)] + [(name, ctypes.c_void_p) for name in (
            "x", "ids", "ranks", "counts", "expert_counts", "expert_offsets", "expert_tasks", "expert_rows",
            "expert_output", "tables", "status")] + [(name, ctypes.c_void_p * EP_MAX_RANKS) for name in (
                "recv_rows_peers", "return_rows_peers", "all_counts_peers", "flags_peers")] + [
        ("expert_chain", ctypes.c_void_p), ("expert_chain_words", ctypes.c_int32), ("reserved2", ctypes.c_int32),
        ("expert_status", ctypes.c_void_p), ("mapping", ctypes.c_void_p),
        ("row_dest_peers", ctypes.c_void_p * EP_MAX_RANKS)]


EXPORTS = {
    "b200moe_abi_version": (ctypes.c_int, []),
    "b200moe_last_error": (ctypes.c_char_p, []),
    "b200moe_plan_create": (ctypes.c_int, [ctypes.POINTER(Shape), ctypes.POINTER(ctypes.c_void_p)]),
    "b200moe_plan_workspace": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(Workspace)]),
    "b200moe_plan_bind": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(Buffers)]),
    "b200moe_forward": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "b200moe_router": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "b200moe_dispatch": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "b200moe_gate_up": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "b200moe_down": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "b200moe_combine": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "b200moe_route": (ctypes.c_int, [ctypes.POINTER(RouteArgs), ctypes.c_void_p]),
    "b200moe_linear_create": (ctypes.c_int, [ctypes.POINTER(LinearShape), ctypes.POINTER(ctypes.c_void_p)]),
    "b200moe_linear_workspace": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(LinearWorkspace)]),
    "b200moe_linear_bind": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(LinearBuffers)]),
    "b200moe_linear_forward": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "b200moe_linear_destroy": (None, [ctypes.c_void_p]),
    "b200moe_dispatch_static": (ctypes.c_int, [ctypes.POINTER(DispatchArgs), ctypes.c_void_p]),
    "b200moe_plan_chain": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p),
                                          ctypes.POINTER(ctypes.c_int32)]),
    "b200moe_ep_table_ints": (ctypes.c_size_t, [ctypes.c_int32, ctypes.c_int32]),
    "b200moe_peer_alloc": (ctypes.c_int, [ctypes.c_size_t, ctypes.POINTER(ctypes.c_void_p)]),
    "b200moe_peer_free": (ctypes.c_int, [ctypes.c_void_p]),
    "b200moe_peer_export": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_char_p]),
    "b200moe_peer_import": (ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p)]),
    "b200moe_peer_close": (ctypes.c_int, [ctypes.c_void_p]),
    "b200moe_ep_exchange_counts": (ctypes.c_int, [ctypes.POINTER(EpArgs), ctypes.c_void_p]),
    "b200moe_ep_send_rows": (ctypes.c_int, [ctypes.POINTER(EpArgs), ctypes.c_void_p]),
    "b200moe_ep_return_rows": (ctypes.c_int, [ctypes.POINTER(EpArgs), ctypes.c_void_p]),
    "b200moe_plan_destroy": (None, [ctypes.c_void_p]),
}

_LIB = None
_LOCK = threading.Lock()


def load():
    """Load the library once; raise if it is absent or has the wrong ABI."""
    global _LIB
    with _LOCK:
        if _LIB is None:
            if not LIBRARY_PATH.is_file():
                raise RuntimeError(
                    f"{LIBRARY_PATH} is missing: build it with `python -m llm_gpu_kernels_b200.build` "
                    "(there is no fallback path)")
            lib = ctypes.CDLL(str(LIBRARY_PATH))
            for name, (restype, argtypes) in EXPORTS.items():
                fn = getattr(lib, name)  # AttributeError if the symbol is not exported
                fn.restype = restype
                fn.argtypes = argtypes
            if lib.b200moe_abi_version() != ABI_VERSION:
                raise RuntimeError("libb200moe.so has an unexpected ABI version")
            _LIB = lib
    return _LIB


def last_error() -> str:
    return load().b200moe_last_error().decode(errors="replace")


def check(code: int):
    """Map a negative return code onto the exception type the reference raises
    for the same condition (ValueError for bad arguments, RuntimeError else)."""
    if code == 0:
        return
    message = last_error()
    if code == ERR_INVALID:
        raise ValueError(message)
    raise RuntimeError(f"b200moe error {code}: {message}")


# bound once: looking the names up at every call would take a quarter longer
_is_compiling = torch.compiler.is_compiling
_dispatch_modes = torch._C._len_torch_dispatch_stack
_function_modes = torch._C._len_torch_function_stack
_jit_tracing = torch._C._is_tracing
_profiling = torch.autograd._profiler_enabled


def tracing():
    """Something records or replaces PyTorch operators: torch.compile, export, torch.jit.trace, make_fx (before dispatch
    by a function mode), a dispatch or function mode, a profiler. Calls of the library must be visible to it as operators;
    a recording that lacks them gives old results for new inputs. A default device is a function mode too, but none of
    these."""
    return (_is_compiling() or _dispatch_modes() > 0 or _jit_tracing() or _profiling()
            or _function_modes() > 0 and not all(isinstance(mode, DeviceContext) for mode in _get_current_function_mode_stack()))


def launch(call, args, device, written):
    """``call(args, stream)`` on the current stream of device ``device``; ``args`` is a struct or a plan handle. The
    tensors ``written`` count as modified in place, so that autograd refuses a backward pass through values that were
    overwritten. Kept short: for one token the kernels behind it take less time than this function."""
    arg = ctypes.byref(args) if isinstance(args, ctypes.Structure) else args
    if torch._C._cuda_getDevice() == device:
        code = call(arg, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            code = call(arg, torch.cuda.current_stream().cuda_stream)
    if code:
        check(code)
    torch._C._increment_version(written)   # torch.autograd.graph.increment_version without its look at the type


def _span(t):
    """First byte and one past the last byte that tensor ``t`` covers."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def check_disjoint(written, read):
    """A tensor that a kernel writes may not share memory with another one it writes or reads."""
    written = [t for t in written if t is not None and t.numel()]
    others = [t for t in read if t is not None and t.numel()]
    for i, w in enumerate(written):
        for t in written[:i] + others:
            a, b = _span(w), _span(t)
            if a[0] < b[1] and b[0] < a[1]:
                raise ValueError("an output shares memory with another output or with an input")
