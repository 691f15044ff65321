"""Layer norm over the last dimensions (csrc/layer_norm.hip).

``torch.nn.functional.layer_norm`` semantics. bf16 or fp32 rows, fp32 weight and bias, statistics in
fp32 over (x - mean). Rows may be slices of wider ones (a channel slice, an ``empty_nhwc`` view
permuted to channels last): any row stride is read in place. Weight and bias gradients are sums in
a fixed order (the same bits every time) and go straight into a live ``.grad`` buffer.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as TF

from .common import (BF16, F32, accumulation_sink, fast_apply, first_derivative_only, lib, native, observed, on_device, ptr,
                     refuse_updated, same_device, stream_handle, track_leaves, updates_seen)


def _rows(t, D):
    """(``t`` as (rows, D) whose rows are dense and do not overlap, row stride); a view where the strides allow."""
    if t.dim() != 2:
        t = t.reshape(-1, D)
    s0, s1 = t.stride()
    rows = t.shape[0]
    if (s1 != 1 and D > 1) or (s0 < D and rows > 1):
        t = t.contiguous()
        s0 = D
    return t, (s0 if rows > 1 else D)


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _forward(x, ld, weight, bias, eps, train):
    """(y, stats) of dense rows x: per-row (mean, 1 / std) where a backward pass is going to need them."""
    rows, D = x.shape
    y = torch.empty((rows, D), dtype=x.dtype, device=x.device)
    stats = torch.empty((rows, 2), dtype=F32, device=x.device) if train else None
    if rows:
        lib().layer_norm_fwd(ptr(x), int(x.dtype == BF16), ld, ptr(weight), ptr(bias), ptr(y), ptr(stats), rows, D, eps,
                             stream_handle())
    return y, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, leaves):  # leaves: the caller's tensors, whose views the others may be
        with on_device(x):
            track_leaves(ctx, *leaves)
            x2, ld = _rows(x, x.shape[-1])
            y, stats = _forward(x2, ld, _dense(weight), _dense(bias), eps, True)
        ctx.seen = updates_seen(weight)
        ctx.save_for_backward(x, weight, bias, stats)
        return y if x.dim() == 2 else y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        return first_derivative_only("layer_norm", _backward, ctx, dy)


def _backward(ctx, dy, sinks):
    # runs on autograd's device thread, where every Python step costs more than in the forward pass
    x, weight, bias, stats = ctx.saved_tensors
    refuse_updated("layer_norm", "weight", weight, ctx.seen)
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dtype = x.dtype
    dx = (torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=dtype, device=x.device)) if need_x else None
    x, ld = _rows(x, x.shape[-1])
    rows, D = x.shape
    if not rows:
        return dx, torch.zeros_like(weight) if need_w else None, torch.zeros_like(bias) if need_b else None, None, None
    g, ldg = _rows(dy if dy.dtype == dtype else dy.to(dtype), D)
    w = _dense(weight)
    sw = accumulation_sink(ctx, 1, weight) if need_w and sinks else None
    sb = accumulation_sink(ctx, 1 if weight is None else 2, bias) if need_b and sinks else None
    dw = sw if sw is not None else x.new_empty(D, dtype=F32) if need_w else None
    db = sb if sb is not None else x.new_empty(D, dtype=F32) if need_b else None
    bf16 = int(dtype == BF16)
    parts = lib().layer_norm_parts(bf16, rows, D)
    part = x.new_empty(parts * 2 * D, dtype=F32) if need_w or need_b else None
    # (the engine runs a node on the device and stream of its forward pass)
    lib().layer_norm_bwd(x.data_ptr(), bf16, ld, g.data_ptr(), ldg, ptr(w), stats.data_ptr(), ptr(dx), ptr(part), parts, ptr(dw),
                         ptr(db), int(sw is not None), int(sb is not None), rows, D, stream_handle())
    return dx, None if sw is not None else dw, None if sb is not None else db, None, None


_apply = fast_apply(_LayerNormFn)


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last ``len(normalized_shape)``
    dimensions of ``x``. On the GPU ``x`` is bf16 or fp32, ``weight`` and ``bias`` fp32 (or None);
    y has x's type. ``eps`` > 0."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    lead = x.dim() - len(shape)
    if not shape or lead < 0 or x.shape[lead:] != shape:
        raise ValueError(f"layer_norm: the last dimensions of an input of shape {tuple(x.shape)} are not {shape}")
    if not 0 < eps < math.inf:
        raise ValueError(f"layer_norm: eps must be positive and finite, got {eps}")
    on_gpu = native(x)
    train = (torch.is_grad_enabled() and x.requires_grad) or observed()
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != shape:
            raise ValueError(f"layer_norm: {name} has shape {tuple(t.shape)}, expected {shape}")
        if on_gpu and t.dtype != F32:
            raise TypeError(f"layer_norm: {name} must be float32, got {t.dtype}")
        train = train or (t.requires_grad and torch.is_grad_enabled())
    same_device("layer_norm", x, weight, bias)
    if not on_gpu:
        w, b = (t.to(x.dtype) if t is not None and x.dtype == torch.float64 else t for t in (weight, bias))
        wide = TF.layer_norm(x if x.dtype == torch.float64 else x.float(), shape, w, b, eps)
        return wide.to(x.dtype)
    if x.dtype != BF16 and x.dtype != F32:
        raise TypeError(f"layer_norm: the input must be bfloat16 or float32, got {x.dtype}")
    D = shape[0] if len(shape) == 1 else math.prod(shape)
    if D == 0:
        raise ValueError("layer_norm: a normalized dimension is empty")
    if not train:
        with on_device(x):
            x2, ld = _rows(x, D)
            y = _forward(x2, ld, _dense(weight), _dense(bias), float(eps), False)[0]
        return y if x.dim() == 2 and lead == 1 else y.view(x.shape)
    leaves = (x, weight, bias)
    if len(shape) > 1:
        x2 = x.reshape(*x.shape[:-len(shape)], D)
        weight, bias = (t.reshape(D) if t is not None else None for t in (weight, bias))
        return _apply(x2, weight, bias, float(eps), leaves).reshape(x.shape)
    return _apply(x, weight, bias, float(eps), leaves)
