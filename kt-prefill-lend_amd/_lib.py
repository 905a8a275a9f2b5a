"""ctypes binding of lib/libktmi.so (the C ABI declared in include/ktmi.h).

The library is loaded once per process; a missing library raises at import of the
first op (there is no CPU fallback). Every wrapper raises RuntimeError with
ktmi_last_error()'s text when a call returns a negative status.
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

LIB_PATH = Path(os.environ.get("KTMI_LIB", Path(__file__).resolve().parent / "lib" / "libktmi.so"))

KTMI_OK = 0
KTMI_F32, KTMI_F16, KTMI_BF16 = 0, 1, 2
W4_DENSE, W4_IDS, W4_SORTED = 0, 1, 2
MODE_AUTO, MODE_GEMV, MODE_GROUPED, MODE_DECODE = 0, 1, 2, 3
STAGE_EVENTS = 6
NOALLOC_SCRATCH_BYTES = 64 << 20  # KTMI_NOALLOC_SCRATCH_BYTES

_i64, _i32, _vp = C.c_int64, C.c_int, C.c_void_p


class ktmi_layer(C.Structure):
    _fields_ = [
        ("hidden", C.c_int64),
        ("inter", C.c_int64),
        ("n_slots", C.c_int64),
        ("type13", C.c_int32),
        ("type2", C.c_int32),
        ("w13", C.c_void_p),
        ("w2", C.c_void_p),
        ("w_is_table", C.c_int32),
        ("reserved", C.c_int32),
    ]


class ktmi_bank(C.Structure):
    _fields_ = [
        ("gate", C.c_void_p),
        ("up", C.c_void_p),
        ("down", C.c_void_p),
        ("part_gate", C.c_int64),
        ("part_up", C.c_int64),
        ("part_down", C.c_int64),
        ("n_experts", C.c_int64),
    ]


class ktmi_w4_kernel(C.Structure):
    _fields_ = [
        ("x_rows", C.c_int32),
        ("col_waves", C.c_int32),
        ("weight_rows", C.c_int32),
        ("tiles", C.c_int32),
        ("staged", C.c_int32),
    ]


# name -> (restype, argtypes); every symbol declared in include/ktmi.h
SIGNATURES = {
    "ktmi_last_error": (C.c_char_p, []),
    "ktmi_version": (_i32, []),
    "ktmi_type_supported": (_i32, [_i32]),
    "ktmi_row_bytes": (_i64, [_i64, _i32]),
    "ktmi_q8_1_row_bytes": (_i64, [_i64]),
    "ktmi_quantize_q8_1": (_i32, [_vp, _i32, _i64, _i64, _vp, _vp]),
    "ktmi_moe_a8_vec_workspace": (_i64, [_i64, _i64]),
    "ktmi_moe_a8_vec": (_i32, [_vp, _i32, _i64, _vp, _i32, _vp, _i64, _i32, _i64, _i64, _i32, _vp, _vp, _i64, _vp]),
    "ktmi_dequant_experts": (_i32, [_vp, _i64, _i32, _i64, _i64, _i64, _vp, _i64, _vp]),
    "ktmi_hot_route": (_i32, [_vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp]),
    "ktmi_silu_and_mul": (_i32, [_vp, _i32, _i64, _i64, _vp, _vp]),
    "ktmi_combine": (_i32, [_vp, _i32, _vp, _i64, _i64, _i64, _vp, _vp]),
    "ktmi_moe_sort_workspace": (_i64, [_i64, _i64, _i64]),
    "ktmi_moe_sort": (_i32, [_vp, _i32, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _vp]),
    "ktmi_moe_unsort": (_i32, [_vp, _i32, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _vp]),
    "ktmi_moe_unsort_grad": (_i32, [_vp, _i64, _vp, _i64, _i32, _i64, _vp, _vp, _i64, _i64, _vp, _vp, _vp]),
    "ktmi_w4_vec": (_i32, [_vp, _i32, _i64, _i64, _vp, _vp, _i32, _vp, _i64, _i64, _i64, _vp, _vp]),
    "ktmi_moe_w4_vec_workspace": (_i64, [_i64, _i64, _i64]),
    "ktmi_moe_w4_vec": (_i32, [_vp, _i32, _i64, _i64, _vp, _vp, _i32, _vp, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _vp,
                               _i64, _vp]),
    "ktmi_moe_w4_sorted": (_i32, [_vp, _i32, _i64, _i64, _vp, _vp, _i32, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _vp]),
    "ktmi_w4_kernel_of": (_i32, [_i32, _i32, _i64, _i64, _i64, _i64, _i64, C.POINTER(ktmi_w4_kernel)]),
    "ktmi_moe_layer_workspace": (_i64, [C.POINTER(ktmi_layer), _i64, _i64, _i32]),
    "ktmi_moe_layer": (_i32, [C.POINTER(ktmi_layer), _vp, _vp, _vp, _i64, _i64, _vp, _vp, _i64, _i32, _vp]),
    "ktmi_moe_layer_mode": (_i32, [C.POINTER(ktmi_layer), _i64, _i64]),
    "ktmi_moe_layer_pass_tokens": (_i64, [C.POINTER(ktmi_layer), _i64]),
    "ktmi_moe_layer_noalloc": (_i32, [C.POINTER(ktmi_layer), _vp, _vp, _vp, _i64, _i64, _vp, _i32, _vp]),
    "ktmi_set_stage_events": (_i32, [C.POINTER(C.c_void_p), _i32]),
    "ktmi_quantize_rows_host": (_i32, [_vp, _i64, _i64, _i32, _vp, _i32]),
    "ktmi_streamer_create": (_vp, [_i64, _i64, _i64, _i32]),
    "ktmi_streamer_destroy": (_i32, [_vp]),
    "ktmi_streamer_slot": (_i32, [_vp, _i32, C.POINTER(C.c_void_p), C.POINTER(C.c_void_p)]),
    "ktmi_streamer_stage": (_i32, [_vp, _i32, C.POINTER(ktmi_bank), _i64, _i64]),
    "ktmi_streamer_acquire": (_i32, [_vp, _i32, _vp]),
    "ktmi_streamer_release": (_i32, [_vp, _i32, _vp]),
    "ktmi_streamer_sync": (_i32, [_vp]),
    "ktmi_streamer_copy_stream": (_vp, [_vp]),
    "ktmi_remap_ids": (_i32, [_vp, _i64, _i32, _i32, _vp, _vp]),
    "ktmi_add_bf16": (_i32, [_vp, _vp, _i64, _vp]),
    "ktmi_host_alloc": (_vp, [_i64]),
    "ktmi_host_free": (_i32, [_vp]),
    "ktmi_cpu_moe_create": (_vp, [_i64, _i64, _i32, _i32, C.POINTER(ktmi_bank), _i32, _i64, _i64]),
    "ktmi_cpu_moe_destroy": (_i32, [_vp]),
    "ktmi_cpu_moe_forward": (_i32, [_vp, _i64, _i64, _vp, _vp, _vp, _vp]),
    "ktmi_cpu_moe_submit": (_i32, [_vp, _vp, _vp, _vp, _i64, _i64, _vp]),
    "ktmi_cpu_moe_sync_add": (_i32, [_vp, _vp, _vp]),
    "ktmi_cpu_moe_threads": (_i32, [_vp]),
    "ktmi_cpu_moe_isa": (C.c_char_p, [_vp]),
    "ktmi_cpu_moe_set_add_wait": (_i32, [_vp, _i64]),
}

_lib = None


def lib():
    """The loaded library; raises if it was not built (there is no fallback)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"ktmi: {LIB_PATH} is missing; build it with kt-prefill-lend_amd/build.py")
        L = C.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def check(rc: int, what: str = "ktmi") -> None:
    if rc != KTMI_OK:
        msg = lib().ktmi_last_error().decode(errors="replace")
        raise RuntimeError(f"{what} failed ({rc}): {msg}")


def ptr(t) -> int:
    """Device (or host) address of a tensor's first element."""
    return t.data_ptr() if t is not None else 0


def stream_ptr(device=None) -> int:
    import torch

    return torch.cuda.current_stream(device).cuda_stream


_torch = None  # what on_device_of takes from torch, bound by its first call (looked up anew it takes 0.5 us a call)


def _bind_torch():
    global _torch
    import torch
    import torch.fx

    c = torch._C
    _torch = torch.autograd.forward_ad, torch.fx._symbolic_trace, c._is_tracing, c._cuda_getDevice, c._cuda_getCurrentRawStream
    return _torch


def _refuse_tangents(what, tensors):
    """Refuses tensors with a forward-mode tangent: the result would have none, that is a derivative of 0."""
    import torch

    for t in tensors:
        if isinstance(t, torch.Tensor) and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative: call it on the primal tensors")


def _refuse_traces(what):
    """Refuses traces of torch's operations: they would hold the outputs' allocations alone."""
    import torch
    from torch.fx.experimental.proxy_tensor import get_proxy_mode  # this thread's

    if torch.jit.is_tracing() or get_proxy_mode() is not None:
        raise RuntimeError(f"{what} cannot be traced: its kernels are no torch operations")


def on_device_of(what, t, fn, *args):
    """fn(stream handle, *args) with t's device current: the current stream of that device, on which the
    call's launches and its tensors' allocations are ordered. what: the call's name in errors."""
    forward_ad, fx, jit_tracing, current_device, stream = _torch or _bind_torch()
    if forward_ad._current_level >= 0:
        _refuse_tangents(what, args)
    if fx._is_fx_tracing_flag or jit_tracing():
        _refuse_traces(what)
    index = t.get_device()
    if current_device() == index:
        return fn(stream(index), *args)
    import torch

    with torch.cuda.device(index):
        return fn(stream(index), *args)


def dtype_code(dtype) -> int:
    import torch

    if dtype == torch.bfloat16:
        return KTMI_BF16
    if dtype == torch.float16:
        return KTMI_F16
    if dtype == torch.float32:
        return KTMI_F32
    raise TypeError(f"ktmi: unsupported activation dtype {dtype}")
