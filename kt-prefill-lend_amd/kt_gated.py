"""Gated and linear products of an expert layer with their gradients, for weights in bf16, f16 or f32.

    h = gated(x, w13)                          dense: w13 [2I, K], rows [gate; up]: h [T, I] = act(x Wg^T) * (x Wu^T)
    h = moe_gated_sorted(rows, w13, offsets)   rows sorted by expert (kt_moe_sort.moe_sort), w13 [E, 2I, K]
    y = moe_linear_sorted(rows, w, offsets)    y[p] = W[e] rows[p], w [E, N, K]

A layer outside the built-in one, trained or served:

    s = moe_sort(x, topk_ids, n_experts)
    y = moe_unsort(moe_linear_sorted(moe_gated_sorted(s.rows, w13, s.offsets), w2, s.offsets), topk_w, s.pos)

Both projections, the activation and the product are one kernel, for single rows too. x and w are of one
type; sums are in fp32 and rounded once to it. act: "silu", or "gelu_tanh" (gelu's tanh form). Rows in no
expert's segment (behind offsets[E]) give zero rows and have zero gradients, whatever they hold.

The gradients, with respect to the rows and the weights: the forward pass keeps x, w13 and both
projections in fp32 (they are not rounded before the activation's derivative takes them); the gradients of the
projections are rounded once to x's type, which is the matrix cores' operand (in f16 one past 65504 is infinite,
and so are the gradients that it enters). No atomics: outputs and gradients are the same from run to run. They are not
differentiable a second time. In fp32 silu and its derivative are right to a few roundings; gelu's sigmoid, whose
argument takes five, is off by up to 2^-15 of itself in its far tail. Forward-mode tangents (NotImplementedError) and
traces by torch.jit.trace or make_fx (RuntimeError) are refused.
All run on the current stream of the tensors' device, allocate from torch's caching allocator, never
synchronise and can be captured into a HIP graph; a captured backward pass needs, as any in torch, that no
graph of the same leaves built outside the capture is alive.
"""
from __future__ import annotations

import torch

from . import _lib
from .kt_moe_sort import _CODES, MAX_EXPERTS, _address, _check_gpu, _rows_of

ACTS = {"silu": _lib.ACT_SILU, "gelu_tanh": _lib.ACT_GELU_TANH}


def _check(what, x, w, offsets, act):
    """Refuses what the kernels do not take; offsets None: dense, act None: no gate."""
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"{what}: x must be [rows, K], got {list(x.shape)}")
    if x.dtype not in _CODES:
        raise TypeError(f"{what}: x must be bfloat16, float16 or float32, got {x.dtype}")
    if w.dtype != x.dtype:
        raise TypeError(f"{what}: w must be x's {x.dtype}, got {w.dtype}")
    lead = 0 if offsets is None else 1
    if w.dim() != 2 + lead or w.shape[-1] != x.shape[1] or w.shape[-2] == 0 or (act is not None and w.shape[-2] % 2):
        raise ValueError(f"{what}: w must be [{'E, ' if lead else ''}{'N' if act is None else '2I'}, {x.shape[1]}], got "
                         f"{list(w.shape)}")
    if act is not None and act not in ACTS:
        raise ValueError(f"{what}: act {act!r} (one of {', '.join(ACTS)})")
    if lead:
        if not 0 < w.shape[0] <= MAX_EXPERTS:
            raise ValueError(f"{what}: {w.shape[0]} experts (1 to {MAX_EXPERTS})")
        if offsets.dtype != torch.int32:
            raise TypeError(f"{what}: offsets must be int32, got {offsets.dtype}")
        if offsets.dim() != 1 or offsets.shape[0] != w.shape[0] + 1:
            raise ValueError(f"{what}: offsets must be [{w.shape[0] + 1}], got {list(offsets.shape)}")
    _check_gpu(what, x, w, offsets)


def _experts(w):
    return w.shape[0] if w.dim() == 3 else 1


def _workspace(what, x, rows, cols, n_experts):
    """(the workspace of such a call or None, its address, its bytes)."""
    need = _lib.lib().ktmi_linear_workspace(what, _CODES[x.dtype], rows, cols, n_experts, x.shape[0])
    if not need:
        return None, None, 0
    ws = x.new_empty((need,), dtype=torch.uint8)
    return ws, ws.data_ptr(), need


def _launch_gated(stream, what, x, w13, offsets, act, keep):
    x, w13 = _rows_of(x), w13.contiguous()
    if offsets is not None:
        offsets = offsets.contiguous()
    R, inter = x.shape[0], w13.shape[-2] // 2
    h = x.new_empty((R, inter))
    sums = x.new_empty((R, 2 * inter), dtype=torch.float32) if keep else None
    ws, at, need = _workspace(_lib.PROD_GATED, x, inter, x.shape[1], _experts(w13))
    rc = _lib.lib().ktmi_gated(x.data_ptr(), _CODES[x.dtype], x.stride(0), x.shape[1], w13.data_ptr(), inter, _experts(w13),
                               None if offsets is None else _address(what, offsets), R, act, h.data_ptr(),
                               sums.data_ptr() if keep else None, at, need, stream)
    if rc:
        _lib.check(rc, what)
    return h, sums


def _launch_linear(stream, what, x, w, offsets):
    x, w, offsets = _rows_of(x), w.contiguous(), offsets.contiguous()
    y = x.new_empty((x.shape[0], w.shape[1]))
    ws, at, need = _workspace(_lib.PROD_LINEAR, x, w.shape[1], w.shape[2], w.shape[0])
    rc = _lib.lib().ktmi_linear(x.data_ptr(), _CODES[x.dtype], x.stride(0), x.shape[1], w.data_ptr(), w.shape[1], w.shape[0],
                                _address(what, offsets), x.shape[0], y.data_ptr(), at, need, stream)
    if rc:
        _lib.check(rc, what)
    return y


def _launch_grads(stream, what, dy, x, w, offsets, want_x, want_w):
    """The gradients of x and w from that of x W^T (by expert)."""
    dy, x, w = _rows_of(dy), _rows_of(x), w.contiguous()
    if offsets is not None:
        offsets = offsets.contiguous()
    L = _lib.lib()
    R, K = x.shape
    N, E, code = w.shape[-2], _experts(w), _CODES[x.dtype]
    at = None if offsets is None else _address(what, offsets)
    dx = x.new_empty((R, K)) if want_x else None
    dw = w.new_empty(w.shape) if want_w else None
    rc = 0
    if want_x:
        ws, ws_at, need = _workspace(_lib.PROD_GRAD_X, x, N, K, E)
        rc = L.ktmi_linear_grad_x(_address(what, dy), code, dy.stride(0), N, w.data_ptr(), K, E, at, R, dx.data_ptr(), ws_at,
                                  need, stream)
    if want_w and not rc:
        ws, ws_at, need = _workspace(_lib.PROD_GRAD_W, x, N, K, E)
        rc = L.ktmi_linear_grad_w(_address(what, dy), code, dy.stride(0), N, x.data_ptr(), x.stride(0), K, E, at, R,
                                  dw.data_ptr(), ws_at, need, stream)
    if rc:
        _lib.check(rc, what)
    return dx, dw


def _launch_gated_grads(stream, what, dh, x, w13, offsets, sums, act, want_x, want_w):
    dh = _rows_of(dh)
    R, inter = dh.shape
    dsums = dh.new_empty((R, 2 * inter))
    rc = _lib.lib().ktmi_gated_grad(sums.data_ptr(), _address(what, dh), _CODES[dh.dtype], dh.stride(0), inter, R, act,
                                    dsums.data_ptr(), stream)
    if rc:
        _lib.check(rc, what)
    return _launch_grads(stream, what, dsums, x, w13, offsets, want_x, want_w)


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, x, w13, offsets, act):
        h, sums = _lib.on_device_of(what, x, _launch_gated, what, x, w13, offsets, act, True)
        ctx.save_for_backward(x, w13, offsets, sums)
        ctx.what, ctx.act = what + "'s gradient", act
        return h

    @staticmethod
    def backward(ctx, dh):
        if torch.is_grad_enabled():
            return _Gated.once(ctx, dh)
        x, w13, offsets, sums = ctx.saved_tensors
        dx, dw = _lib.on_device_of(ctx.what, dh, _launch_gated_grads, ctx.what, dh, x, w13, offsets, sums, ctx.act,
                                   ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        return None, dx, dw, None, None

    # of a graph for second derivatives: the same without a graph of its own, refused when one is asked for
    once = staticmethod(torch.autograd.function.once_differentiable(lambda ctx, dh: _Gated.backward(ctx, dh)))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, x, w, offsets):
        y = _lib.on_device_of(what, x, _launch_linear, what, x, w, offsets)
        ctx.save_for_backward(x, w, offsets)
        ctx.what = what + "'s gradient"
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            return _Linear.once(ctx, dy)
        x, w, offsets = ctx.saved_tensors
        dx, dw = _lib.on_device_of(ctx.what, dy, _launch_grads, ctx.what, dy, x, w, offsets, ctx.needs_input_grad[1],
                                   ctx.needs_input_grad[2])
        return None, dx, dw, None

    once = staticmethod(torch.autograd.function.once_differentiable(lambda ctx, dy: _Linear.backward(ctx, dy)))


def _run_gated(what, x, w13, offsets, act):
    _check(what, x, w13, offsets, act)
    if torch.is_grad_enabled() and (x.requires_grad or w13.requires_grad):
        return _Gated.apply(what, x, w13, offsets, ACTS[act])
    return _lib.on_device_of(what, x, _launch_gated, what, x, w13, offsets, ACTS[act], False)[0]


def gated(x: torch.Tensor, w13: torch.Tensor, act: str = "silu") -> torch.Tensor:
    """h [T, I] = act(x Wg^T) * (x Wu^T) for x [T, K] and w13 [2I, K] = rows [gate; up]. Differentiable in both."""
    return _run_gated("gated", x, w13, None, act)


def moe_gated_sorted(rows: torch.Tensor, w13: torch.Tensor, offsets: torch.Tensor, act: str = "silu") -> torch.Tensor:
    """h [R, I] for rows [R, K] sorted by expert and w13 [E, 2I, K]: expert e's rows are [offsets[e], offsets[e + 1])
    (int32 [E + 1], ascending, as moe_sort gives them); rows past offsets[E] give zero rows. Differentiable in the
    rows and in w13."""
    if offsets is None:
        raise TypeError("moe_gated_sorted: offsets must be int32, got None")
    return _run_gated("moe_gated_sorted", rows, w13, offsets, act)


def moe_linear_sorted(rows: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """y [R, N] for rows [R, K] sorted by expert and w [E, N, K], rows and offsets as for moe_gated_sorted.
    Differentiable in the rows and in w."""
    if offsets is None:
        raise TypeError("moe_linear_sorted: offsets must be int32, got None")
    what = "moe_linear_sorted"
    _check(what, rows, w, offsets, None)
    if torch.is_grad_enabled() and (rows.requires_grad or w.requires_grad):
        return _Linear.apply(what, rows, w, offsets)
    return _lib.on_device_of(what, rows, _launch_linear, what, rows, w, offsets)
