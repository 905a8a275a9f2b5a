"""Tokens sorted by expert and back, with the route weights applied, and the gradients of both.

For expert products outside the built-in layer (`kt_gguf_hot.moe_layer`): other weight formats
(`kt_w4_vec.moe_w4_sorted`, which has no gradient), adapters, ranks that hold part of the experts,
training.

    s = moe_sort(x, topk_ids, n_experts)          # s.rows[s.offsets[e]:s.offsets[e + 1]] are expert e's
    y = moe_unsort(experts(s.rows), topk_w, s.pos)  # the weighted sum over each token's routes

Routes whose id lies outside [0, n_experts) (-1: an expert on the CPU or on another rank) belong to
no expert: their rows come last and are zero, and add nothing on the way back. The order is stable
(by expert, then by route), so every output and gradient is the same from run to run; sums are in
fp32 and rounded once. Both run on the current stream of the tensors' device, allocate from torch's
caching allocator, never synchronise and can be captured into a HIP graph. A captured backward pass
needs, as any in torch, that no graph of the same leaves built outside the capture is alive.

The gradients: of moe_sort with respect to x (the sum of its routes' rows), of moe_unsort with
respect to the rows and the weights. They are not differentiable a second time. Forward-mode tangents
(NotImplementedError) and traces by torch.jit.trace or make_fx (RuntimeError) are refused.
"""
from __future__ import annotations

from collections import namedtuple

import torch

from . import _lib

MAX_EXPERTS = 2048

# rows [T*k, K] in x's type; offsets int32 [n_experts + 1]; perm int32 [T*k], the route at each place (its
# complement past offsets[-1]); pos int32 [T, k], the place of each route (its complement without an expert)
MoeSorted = namedtuple("MoeSorted", ["rows", "offsets", "perm", "pos"])

_CODES = {torch.float32: _lib.KTMI_F32, torch.float16: _lib.KTMI_F16, torch.bfloat16: _lib.KTMI_BF16}


def _rows_of(t):
    """t with its values of a row next to each other and rows that do not overlap."""
    return t if t.is_contiguous() or (t.stride(1) == 1 and t.stride(0) >= t.shape[1]) else t.contiguous()


def _address(what, t):
    """t's first element, where the library takes a null pointer for an argument left out."""
    p = t.data_ptr()
    if p == 0 and t.numel():
        raise TypeError(f"{what}: a {type(t).__name__} holds no memory of its own: pass its local tensor")
    return p


def _check_gpu(what, *tensors):
    """Refuses tensors that are not all on one GPU (None: an argument left out)."""
    index = tensors[0].get_device()  # -1 on the CPU
    for t in tensors:
        if t is not None and (index < 0 or t.get_device() != index):
            raise ValueError(f"{what}: tensors must be on one GPU, got {tensors[0].device} and {t.device}")


def _check_sort(x, ids, n_experts):
    if x.dim() != 2 or ids.dim() != 2 or ids.shape[0] != x.shape[0] or ids.shape[1] == 0 or x.shape[1] == 0:
        raise ValueError(f"moe_sort: x must be [T, K] and ids [T, k], got {list(x.shape)} and {list(ids.shape)}")
    if x.dtype not in _CODES:
        raise TypeError(f"moe_sort: x must be bfloat16, float16 or float32, got {x.dtype}")
    if ids.dtype != torch.int32:
        raise TypeError(f"moe_sort: ids must be int32, got {ids.dtype}")
    if not 0 < n_experts <= MAX_EXPERTS:
        raise ValueError(f"moe_sort: {n_experts} experts (1 to {MAX_EXPERTS})")
    _check_gpu("moe_sort", x, ids)


def _check_unsort(rows, topk_w, pos):
    if rows.dim() != 2 or pos.dim() != 2 or rows.shape[0] != pos.numel() or pos.shape[1] == 0 or rows.shape[1] == 0:
        raise ValueError(f"moe_unsort: rows must be [T*k, K] and pos [T, k], got {list(rows.shape)} and {list(pos.shape)}")
    if rows.dtype not in _CODES:
        raise TypeError(f"moe_unsort: rows must be bfloat16, float16 or float32, got {rows.dtype}")
    if pos.dtype != torch.int32:
        raise TypeError(f"moe_unsort: pos must be int32, got {pos.dtype}")
    if topk_w is not None:
        if topk_w.dtype != torch.float32:
            raise TypeError(f"moe_unsort: topk_w must be float32, got {topk_w.dtype}")
        if topk_w.shape != pos.shape:
            raise ValueError(f"moe_unsort: topk_w is {list(topk_w.shape)}, pos {list(pos.shape)}")
    _check_gpu("moe_unsort", rows, topk_w, pos)


def _launch_sort(stream, x, ids, n_experts):
    L = _lib.lib()
    T, K = x.shape
    k = ids.shape[1]
    x, ids = _rows_of(x), ids.contiguous()
    rows = x.new_empty((T * k, K))
    offsets = ids.new_empty((n_experts + 1,))
    perm = ids.new_empty((T * k,))
    pos = ids.new_empty((T, k))
    need = L.ktmi_moe_sort_workspace(T, k, n_experts)
    ws = ids.new_empty((need,), dtype=torch.uint8) if need else None
    rc = L.ktmi_moe_sort(_address("moe_sort", x), _CODES[x.dtype], x.stride(0), K, ids.data_ptr(), T, k, n_experts,
                         rows.data_ptr(), offsets.data_ptr(), perm.data_ptr(), pos.data_ptr(),
                         ws.data_ptr() if need else None, need, stream)
    if rc:
        _lib.check(rc, "moe_sort")
    return rows, offsets, perm, pos


def _launch_unsort(stream, rows, topk_w, pos):
    T, k = pos.shape
    K = rows.shape[1]
    rows, pos = _rows_of(rows), pos.contiguous()
    if topk_w is not None:
        topk_w = topk_w.contiguous()
    y = rows.new_empty((T, K))
    rc = _lib.lib().ktmi_moe_unsort(rows.data_ptr(), _CODES[rows.dtype], rows.stride(0), K,
                                    None if topk_w is None else _address("moe_unsort", topk_w), pos.data_ptr(), T, k,
                                    y.data_ptr(), stream)
    if rc:
        _lib.check(rc, "moe_unsort")
    return y


def _launch_unsort_grad(stream, dy, rows, topk_w, pos, want_rows, want_w):
    T, k = pos.shape
    K = dy.shape[1]
    dy, pos = _rows_of(dy), pos.contiguous()
    rows = _rows_of(rows) if want_w else None
    if topk_w is not None:
        topk_w = topk_w.contiguous()
    drows = dy.new_empty((T * k, K)) if want_rows else None
    dw = dy.new_empty((T, k), dtype=torch.float32) if want_w else None
    what = "moe_unsort's gradient"
    rc = _lib.lib().ktmi_moe_unsort_grad(_address(what, dy), dy.stride(0), rows.data_ptr() if want_w else None,
                                         rows.stride(0) if want_w else K, _CODES[dy.dtype], K,
                                         None if topk_w is None else _address(what, topk_w), pos.data_ptr(), T, k,
                                         drows.data_ptr() if want_rows else None, dw.data_ptr() if want_w else None,
                                         stream)
    if rc:
        _lib.check(rc, "moe_unsort_grad")
    return drows, dw


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, n_experts):
        rows, offsets, perm, pos = _lib.on_device_of("moe_sort", x, _launch_sort, x, ids, n_experts)
        ctx.save_for_backward(pos)
        ctx.mark_non_differentiable(offsets, perm, pos)
        ctx.set_materialize_grads(False)
        return rows, offsets, perm, pos

    @staticmethod
    def backward(ctx, drows, *ignored):
        if torch.is_grad_enabled():
            return _Sort.once(ctx, drows, *ignored)
        if drows is None:
            return None, None, None
        pos, = ctx.saved_tensors
        return _lib.on_device_of("moe_sort's gradient", drows, _launch_unsort, drows, None, pos), None, None

    # of a graph for second derivatives: the same without a graph of its own, refused when one is asked for
    once = staticmethod(torch.autograd.function.once_differentiable(lambda ctx, *grads: _Sort.backward(ctx, *grads)))


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, topk_w, pos):
        want_w = topk_w is not None and ctx.needs_input_grad[1]
        ctx.save_for_backward(rows if want_w else None, topk_w, pos)
        return _lib.on_device_of("moe_unsort", rows, _launch_unsort, rows, topk_w, pos)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            return _Unsort.once(ctx, dy)
        rows, topk_w, pos = ctx.saved_tensors
        return (*_lib.on_device_of("moe_unsort's gradient", dy, _launch_unsort_grad, dy, rows, topk_w, pos,
                                   ctx.needs_input_grad[0], rows is not None), None)

    once = staticmethod(torch.autograd.function.once_differentiable(lambda ctx, dy: _Unsort.backward(ctx, dy)))


def moe_sort(x: torch.Tensor, ids: torch.Tensor, n_experts: int) -> MoeSorted:
    """The rows of x [T, K] (bf16, f16 or f32) copied to each of their routes' places: ids int32 [T, k],
    at most 2048 experts, k at most 65535, fewer than 2^31 routes. Returns MoeSorted; differentiable in x."""
    _check_sort(x, ids, n_experts)
    if x.requires_grad and torch.is_grad_enabled():
        return MoeSorted(*_Sort.apply(x, ids, n_experts))
    return MoeSorted(*_lib.on_device_of("moe_sort", x, _launch_sort, x, ids, n_experts))


def moe_unsort(rows: torch.Tensor, topk_w, pos: torch.Tensor) -> torch.Tensor:
    """y[t] = sum over k of topk_w[t, k] * rows[pos[t, k]], [T, K] in the rows' type: rows [T*k, K] in the
    order of moe_sort, topk_w fp32 [T, k] or None (weights 1), pos its pos, which names every row once (so
    that the rows' gradient is written whole). Differentiable in rows and topk_w."""
    _check_unsort(rows, topk_w, pos)
    if torch.is_grad_enabled() and (rows.requires_grad or (topk_w is not None and topk_w.requires_grad)):
        return _Unsort.apply(rows, topk_w, pos)
    return _lib.on_device_of("moe_unsort", rows, _launch_unsort, rows, topk_w, pos)
