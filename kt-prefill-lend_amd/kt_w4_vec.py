"""Products of a few rows with 4-bit weights and group scales, for decode windows.

For checkpoints of plain 4-bit codes with a scale (and zero point) for each group of values along a
row, beside the ggml types of `kt_gguf_moe_multi`:

    y[r, n] = sum_g scales[n, g] * sum_{c in group g} (code[n, c] - zero[n, g]) * x[r, c]

    w4_vec(x, codes, scales)                          dense: codes [N, ceil(K/2)]
    moe_w4_vec(x, codes, scales, ids, top_k)          by route, codes [E, N, ceil(K/2)] (moe_a8_vec_multi's contract)
    moe_w4_sorted(rows, codes, scales, offsets)       rows sorted by expert (kt_moe_sort.moe_sort)

codes: uint8, byte j of a row holds code 2j in its low and code 2j + 1 in its high four bits, or the
same bytes as int32 [.., K/8]; scales: bf16, f16 or f32 [.., ceil(K/group_size)]; zeros: uint8 of that
shape, or None for 8 everywhere; group_size: 32, 64, a multiple of 128, or at least K (one group a
row). x: bf16, f16 or f32; the weights' values are exact, sums are in fp32 and rounded once to x's
type (of f32 x the bits below 2^-133 may be left out). Any K and N (to 2^24), at most 2^23 rows of y.
They run on the current stream of x's device, allocate from torch's caching allocator, never
synchronise and can be captured into a HIP graph. No gradient: inputs that require one are refused
while gradients are recorded (RuntimeError), inputs with a forward-mode tangent always
(NotImplementedError), and so are traces by torch.jit.trace or make_fx (RuntimeError).
"""
from __future__ import annotations

import torch

from . import _lib
from .kt_moe_sort import _CODES, MAX_EXPERTS, _address, _check_gpu, _rows_of


def _check(what, x, codes, scales, zeros, group, lead):
    """Refuses what the kernels do not take; lead: the dimensions before [N, ..] (0 or 1)."""
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"{what}: x must be [rows, K], got {list(x.shape)}")
    if x.dtype not in _CODES:
        raise TypeError(f"{what}: x must be bfloat16, float16 or float32, got {x.dtype}")
    if scales.dtype not in _CODES:
        raise TypeError(f"{what}: scales must be bfloat16, float16 or float32, got {scales.dtype}")
    if codes.dtype not in (torch.uint8, torch.int32):
        raise TypeError(f"{what}: codes must be uint8 or int32, got {codes.dtype}")
    K = x.shape[1]
    if not isinstance(group, int) or group <= 0 or not (group in (32, 64) or group % 128 == 0 or group >= K):
        raise ValueError(f"{what}: group_size {group} (32, 64, a multiple of 128, or at least K = {K})")
    per = 2 if codes.dtype == torch.uint8 else 8
    width, groups = -(-K // per), -(-K // group)
    *front, last = codes.shape
    if len(front) != 1 + lead or last != width or (per == 8 and K % 8) or front[-1] == 0:
        raise ValueError(f"{what}: codes must be {'[E, N, ' if lead else '[N, '}{width}] for K = {K}, got {codes.dtype} "
                         f"{list(codes.shape)}")
    if lead and not 0 < front[0] <= MAX_EXPERTS:
        raise ValueError(f"{what}: {front[0]} experts (1 to {MAX_EXPERTS})")
    want = (*front, groups)
    if scales.shape != want:
        raise ValueError(f"{what}: scales must be {list(want)}, got {list(scales.shape)}")
    if zeros is not None:
        if zeros.dtype != torch.uint8:
            raise TypeError(f"{what}: zeros must be uint8, got {zeros.dtype}")
        if zeros.shape != want:
            raise ValueError(f"{what}: zeros must be {list(want)}, got {list(zeros.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or scales.requires_grad):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _args(x, codes, scales, zeros, group):
    """The contiguous tensors of a call (kept alive by the caller) and the C arguments from x to group."""
    x, codes, scales = _rows_of(x), codes.contiguous(), scales.contiguous()
    group = min(group, x.shape[1])  # one group a row, however large the size that says so
    zeros = None if zeros is None else zeros.contiguous()
    return (x, codes, scales, zeros), (x.data_ptr(), _CODES[x.dtype], x.stride(0), x.shape[1], codes.data_ptr(),
                                       scales.data_ptr(), _CODES[scales.dtype],
                                       None if zeros is None else _address("zeros", zeros), group)


def _launch_dense(stream, x, codes, scales, zeros, group):
    keep, args = _args(x, codes, scales, zeros, group)
    T, N = x.shape[0], codes.shape[0]
    y = x.new_empty((T, N))
    rc = _lib.lib().ktmi_w4_vec(*args, N, T, y.data_ptr(), stream)
    if rc:
        _lib.check(rc, "w4_vec")
    return y


def _launch_routed(stream, x, codes, scales, ids, top_k, zeros, group):
    keep, args = _args(x, codes, scales, zeros, group)
    ids = ids.contiguous()
    T, (E, N) = x.shape[0], codes.shape[:2]
    L = _lib.lib()
    y = x.new_empty((T * top_k, N))
    need = L.ktmi_moe_w4_vec_workspace(T, top_k, E)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    rc = L.ktmi_moe_w4_vec(*args, N, E, ids.data_ptr(), top_k, T, y.data_ptr(), ws.data_ptr() if need else None, need,
                           stream)
    if rc:
        _lib.check(rc, "moe_w4_vec")
    return y


def _launch_sorted(stream, rows, codes, scales, offsets, zeros, group):
    keep, args = _args(rows, codes, scales, zeros, group)
    offsets = offsets.contiguous()
    R, (E, N) = rows.shape[0], codes.shape[:2]
    y = rows.new_empty((R, N))
    rc = _lib.lib().ktmi_moe_w4_sorted(*args, N, E, offsets.data_ptr(), R, y.data_ptr(), stream)
    if rc:
        _lib.check(rc, "moe_w4_sorted")
    return y


def w4_vec(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros=None, group_size: int = 128) -> torch.Tensor:
    """y [T, N] = x W^T for x [T, K] and one matrix, codes [N, ceil(K/2)]; made for up to 64 rows of x."""
    _check("w4_vec", x, codes, scales, zeros, group_size, 0)
    _check_gpu("w4_vec", x, codes, scales, zeros)
    return _lib.on_device_of("w4_vec", x, _launch_dense, x, codes, scales, zeros, group_size)


def moe_w4_vec(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, ids: torch.Tensor, top_k: int, zeros=None,
               group_size: int = 128) -> torch.Tensor:
    """Y [T*top_k, N]: route p = t*top_k + k uses row t of x [T, K] and the matrix of expert ids[p] (int32,
    T*top_k of them); ids outside [0, E) give zero rows. The routes of one expert share one read of its
    weights."""
    _check("moe_w4_vec", x, codes, scales, zeros, group_size, 1)
    if ids.dtype != torch.int32:
        raise TypeError(f"moe_w4_vec: ids must be int32, got {ids.dtype}")
    if not 0 < top_k <= 65535 or ids.numel() != x.shape[0] * top_k:
        raise ValueError(f"moe_w4_vec: {ids.numel()} ids for {x.shape[0]} rows of x and top_k {top_k}")
    _check_gpu("moe_w4_vec", x, codes, scales, zeros, ids)
    return _lib.on_device_of("moe_w4_vec", x, _launch_routed, x, codes, scales, ids, top_k, zeros, group_size)


def moe_w4_sorted(rows: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, offsets: torch.Tensor, zeros=None,
                  group_size: int = 128) -> torch.Tensor:
    """Y [R, N] for rows [R, K] sorted by expert: expert e's are [offsets[e], offsets[e + 1]) (int32 [E + 1],
    ascending, as moe_sort gives them); rows past offsets[E] give zero rows."""
    _check("moe_w4_sorted", rows, codes, scales, zeros, group_size, 1)
    if offsets.dtype != torch.int32:
        raise TypeError(f"moe_w4_sorted: offsets must be int32, got {offsets.dtype}")
    if offsets.dim() != 1 or offsets.shape[0] != codes.shape[0] + 1:
        raise ValueError(f"moe_w4_sorted: offsets must be [{codes.shape[0] + 1}], got {list(offsets.shape)}")
    _check_gpu("moe_w4_sorted", rows, codes, scales, zeros, offsets)
    return _lib.on_device_of("moe_w4_sorted", rows, _launch_sorted, rows, codes, scales, offsets, zeros, group_size)
