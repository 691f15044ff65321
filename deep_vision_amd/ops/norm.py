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

from .common import BF16, F32, accumulation_sink, lib, native, on_device, ptr, same_device, stream_handle, track_leaves


def _rows(t, D):
    """``t`` as (rows, D) whose rows are dense and do not overlap; a view where the strides allow."""
    t = t.reshape(-1, D)
    if (D > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < D):
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else D)


def _forward(x, weight, bias, eps, stats):
    """(y, stats): per-row (mean, 1 / std) where a backward pass is going to need them."""
    D = x.shape[-1]
    x2, ld = _rows(x, D)
    rows = x2.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((rows, 2), dtype=F32, device=x.device) if stats else None
    w, b = (t.detach().contiguous() if t is not None else None for t in (weight, bias))
    if rows:
        with on_device(x):
            lib().layer_norm_fwd(ptr(x2), int(x.dtype == BF16), ld, ptr(w), ptr(b), ptr(y), ptr(stats), rows, D, eps,
                                 stream_handle())
    return y, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        with on_device(x):
            track_leaves(ctx, x, weight, bias)
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        D = x.shape[-1]
        x2, ld = _rows(x, D)
        g, ldg = _rows(dy if dy.dtype == x.dtype else dy.to(x.dtype), D)
        rows, bf16 = x2.shape[0], int(x.dtype == BF16)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        if not rows:
            return (dx, torch.zeros_like(weight) if need_w else None, torch.zeros_like(bias) if need_b else None, None)
        sinks = [accumulation_sink(ctx, i, t) if need else None
                 for i, t, need in ((1, weight, need_w), (2, bias, need_b))]
        dw, db = (s if s is not None else torch.empty(D, dtype=F32, device=x.device) if need else None
                  for s, need in zip(sinks, (need_w, need_b)))
        w = weight.detach().contiguous() if weight is not None else None
        parts = lib().layer_norm_parts(bf16, rows, D)
        part = torch.empty((parts, 2, D), dtype=F32, device=x.device) if need_w or need_b else None
        with on_device(x):
            lib().layer_norm_bwd(ptr(x2), bf16, ld, ptr(g), ldg, ptr(w), ptr(stats), ptr(dx), ptr(part), parts, ptr(dw),
                                 ptr(db), int(sinks[0] is not None), int(sinks[1] is not None), rows, D, stream_handle())
        dw, db = (None if s is not None or t is None else t for s, t in zip(sinks, (dw, db)))
        return dx, dw, db, None


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last ``len(normalized_shape)``
    dimensions of ``x``. On the GPU ``x`` is bf16 or fp32, ``weight`` and ``bias`` fp32 (or None);
    y has x's type. ``eps`` > 0."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(int(n) for n in normalized_shape)
    if not shape or tuple(x.shape[-len(shape):]) != shape or len(shape) > x.dim():
        raise ValueError(f"layer_norm: the last dimensions of an input of shape {tuple(x.shape)} are not {shape}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != shape:
            raise ValueError(f"layer_norm: {name} has shape {tuple(t.shape)}, expected {shape}")
    if not eps > 0 or not math.isfinite(eps):
        raise ValueError(f"layer_norm: eps must be positive and finite, got {eps}")
    same_device("layer_norm", x, weight, bias)
    if not native(x):
        w, b = (t.to(x.dtype) if t is not None and x.dtype == torch.float64 else t for t in (weight, bias))
        wide = TF.layer_norm(x if x.dtype == torch.float64 else x.float(), shape, w, b, eps)
        return wide.to(x.dtype)
    if x.dtype not in (BF16, F32):
        raise TypeError(f"layer_norm: the input must be bfloat16 or float32, got {x.dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dtype != F32:
            raise TypeError(f"layer_norm: {name} must be float32, got {t.dtype}")
    D = math.prod(shape)
    if D == 0:
        raise ValueError("layer_norm: a normalized dimension is empty")
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias))):
        if len(shape) > 1:
            x = x.reshape(*x.shape[:-len(shape)], D)
        return _forward(x, weight, bias, float(eps), False)[0].reshape(*x.shape[:-1], *shape)
    if len(shape) > 1:
        x2 = x.reshape(*x.shape[:-len(shape)], D)
        weight, bias = (t.reshape(D) if t is not None else None for t in (weight, bias))
        return _LayerNormFn.apply(x2, weight, bias, float(eps)).reshape(x.shape)
    return _LayerNormFn.apply(x, weight, bias, float(eps))
