"""Products in 8-bit floating point with a scale for each block of 128, for checkpoints of e4m3 weights.

    y[r, n] = sum_g xs[r, g] * scales[n // 128, g] * sum_{c in block g of 128 columns} xq[r, c] * w[n, c]

    fp8_linear(x, w, scales)                    dense: w [N, K], scales [ceil(N/128), ceil(K/128)]
    moe_fp8_vec(x, w, scales, ids, top_k)       by route, w [E, N, K] (moe_a8_vec_multi's contract)
    moe_fp8_sorted(rows, w, scales, offsets)    rows sorted by expert (kt_moe_sort.moe_sort)

w: float8_e4m3fn (or its bytes as uint8), scales: f32. x: bf16, f16 or f32, quantised on the way for
each row and block of 128 columns: a = max(|x|, 2^-116), xq = e4m3(f32(x * f32(448 / a))), xs = f32(a / 448),
to nearest, ties to even; a value that is not finite makes its row of y NaN. Sums are in fp32 (of y in 16
bits a block's sum by the matrix cores' 8-bit products, which keep about 16 bits below the largest product)
and rounded once to x's type; the two scales' product is an fp32 number (below 2^-126 in its subnormal
steps, past fp32's largest number that one, unless the scale of w is not finite). Any K and N (to 2^24).
They run on the current stream of x's device, allocate from torch's caching allocator, never
synchronise and can be captured into a HIP graph. No gradient: inputs that require one are refused
while gradients are recorded (RuntimeError), inputs with a forward-mode tangent always
(NotImplementedError), and so are traces by torch.jit.trace or make_fx (RuntimeError).
"""
from __future__ import annotations

import torch

from . import _lib
from .kt_moe_sort import _CODES, MAX_EXPERTS, _check_gpu, _rows_of

BLOCK = 128


def _check(what, x, w, scales, lead):
    """Refuses what the kernels do not take; lead: the dimensions before [N, K] (0 or 1)."""
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"{what}: x must be [rows, K], got {list(x.shape)}")
    if x.dtype not in _CODES:
        raise TypeError(f"{what}: x must be bfloat16, float16 or float32, got {x.dtype}")
    if w.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise TypeError(f"{what}: w must be float8_e4m3fn or uint8, got {w.dtype}")
    if scales.dtype != torch.float32:
        raise TypeError(f"{what}: scales must be float32, got {scales.dtype}")
    K = x.shape[1]
    if w.dim() != 2 + lead or w.shape[-1] != K or w.shape[-2] == 0:
        raise ValueError(f"{what}: w must be {'[E, N, ' if lead else '[N, '}{K}], got {list(w.shape)}")
    if lead and not 0 < w.shape[0] <= MAX_EXPERTS:
        raise ValueError(f"{what}: {w.shape[0]} experts (1 to {MAX_EXPERTS})")
    want = (*w.shape[:-2], -(-w.shape[-2] // BLOCK), -(-K // BLOCK))
    if scales.shape != want:
        raise ValueError(f"{what}: scales must be {list(want)}, got {list(scales.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or scales.requires_grad or w.requires_grad):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _launch_dense(stream, x, w, scales):
    x, w, scales = _rows_of(x), w.contiguous(), scales.contiguous()
    L = _lib.lib()
    T, K = x.shape
    N = w.shape[0]
    y = x.new_empty((T, N))
    need = L.ktmi_fp8_linear_workspace(N, K, T)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    rc = L.ktmi_fp8_linear(x.data_ptr(), _CODES[x.dtype], x.stride(0), K, w.data_ptr(), scales.data_ptr(), N, T, y.data_ptr(),
                           ws.data_ptr() if need else None, need, stream)
    if rc:
        _lib.check(rc, "fp8_linear")
    return y


def _launch_routed(stream, x, w, scales, ids, top_k):
    x, w, scales, ids = _rows_of(x), w.contiguous(), scales.contiguous(), ids.contiguous()
    L = _lib.lib()
    T, K = x.shape
    E, N = w.shape[:2]
    y = x.new_empty((T * top_k, N))
    need = L.ktmi_moe_fp8_vec_workspace(N, K, T, top_k, E)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    rc = L.ktmi_moe_fp8_vec(x.data_ptr(), _CODES[x.dtype], x.stride(0), K, w.data_ptr(), scales.data_ptr(), N, E,
                            ids.data_ptr(), top_k, T, y.data_ptr(), ws.data_ptr() if need else None, need, stream)
    if rc:
        _lib.check(rc, "moe_fp8_vec")
    return y


def _launch_sorted(stream, rows, w, scales, offsets):
    rows, w, scales, offsets = _rows_of(rows), w.contiguous(), scales.contiguous(), offsets.contiguous()
    L = _lib.lib()
    R, K = rows.shape
    E, N = w.shape[:2]
    y = rows.new_empty((R, N))
    need = L.ktmi_moe_fp8_sorted_workspace(N, K, E, R)
    ws = rows.new_empty((need,), dtype=torch.uint8) if need else None
    rc = L.ktmi_moe_fp8_sorted(rows.data_ptr(), _CODES[rows.dtype], rows.stride(0), K, w.data_ptr(), scales.data_ptr(), N, E,
                               offsets.data_ptr(), R, y.data_ptr(), ws.data_ptr() if need else None, need, stream)
    if rc:
        _lib.check(rc, "moe_fp8_sorted")
    return y


def fp8_linear(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """y [T, N] = x W^T for x [T, K] and one matrix, w [N, K] with scales [ceil(N/128), ceil(K/128)]."""
    _check("fp8_linear", x, w, scales, 0)
    _check_gpu("fp8_linear", x, w, scales)
    return _lib.on_device_of("fp8_linear", x, _launch_dense, x, w, scales)


def moe_fp8_vec(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, ids: torch.Tensor, top_k: int) -> torch.Tensor:
    """Y [T*top_k, N]: route p = t*top_k + k uses row t of x [T, K] and the matrix of expert ids[p] (int32,
    T*top_k of them); ids outside [0, E) give zero rows. The routes of one expert share one read of its
    weights."""
    _check("moe_fp8_vec", x, w, scales, 1)
    if ids.dtype != torch.int32:
        raise TypeError(f"moe_fp8_vec: ids must be int32, got {ids.dtype}")
    if not 0 < top_k <= 65535 or ids.numel() != x.shape[0] * top_k:
        raise ValueError(f"moe_fp8_vec: {ids.numel()} ids for {x.shape[0]} rows of x and top_k {top_k}")
    _check_gpu("moe_fp8_vec", x, w, scales, ids)
    return _lib.on_device_of("moe_fp8_vec", x, _launch_routed, x, w, scales, ids, top_k)


def moe_fp8_sorted(rows: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Y [R, N] for rows [R, K] sorted by expert: expert e's are [offsets[e], offsets[e + 1]) (int32 [E + 1],
    ascending, as moe_sort gives them); rows past offsets[E] give zero rows."""
    _check("moe_fp8_sorted", rows, w, scales, 1)
    if offsets.dtype != torch.int32:
        raise TypeError(f"moe_fp8_sorted: offsets must be int32, got {offsets.dtype}")
    if offsets.dim() != 1 or offsets.shape[0] != w.shape[0] + 1:
        raise ValueError(f"moe_fp8_sorted: offsets must be [{w.shape[0] + 1}], got {list(offsets.shape)}")
    _check_gpu("moe_fp8_sorted", rows, w, scales, offsets)
    return _lib.on_device_of("moe_fp8_sorted", rows, _launch_sorted, rows, w, scales, offsets)
