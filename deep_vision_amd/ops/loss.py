"""Fused softmax cross-entropy (csrc/loss_optim.hip).

Matches ``nn.CrossEntropyLoss()`` (mean reduction) used by every PT classifier of the
reference (R/ResNet/pytorch/train.py:358). The gradient is produced in the forward launch.
"""
from __future__ import annotations

import torch
import torch.nn.functional as TF

from . import wcache
from .common import (BF16, F32, accumulation_sink, fast_apply, first_derivative_only, lib, native, observed, on_device, ptr,
                     refuse_updated, same_device, stream_handle, track_leaves, updates_seen)


class _XentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, label_smoothing):
        B, C = logits.shape
        lr = torch.empty(B, dtype=F32, device=logits.device)
        need_grad = logits.requires_grad
        grad = torch.empty_like(logits) if need_grad else None
        lib().softmax_xent(ptr(logits), int(logits.dtype == BF16), ptr(labels), B, C, ptr(lr), ptr(grad), 1.0 / B,
                           float(label_smoothing), stream_handle())
        ctx.save_for_backward(grad)
        return lr.mean()  # one reduction launch (sum and scale fused)

    @staticmethod
    def backward(ctx, go):
        (grad,) = ctx.saved_tensors
        if go is None:
            return grad, None, None
        # out of place: the saved buffer stays the unscaled gradient, so a second backward through
        # a retained graph scales the same values again (an in-place mul_ would have returned
        # grad*go1*go2); the scale is read on the device by one native launch
        go = go.detach().to(F32).reshape(1).contiguous()
        out = torch.empty_like(grad)
        lib().scale_by(ptr(grad), ptr(out), grad.numel(), int(grad.dtype == BF16), ptr(go), stream_handle())
        return out, None, None


def cross_entropy(logits, labels, label_smoothing=0.0):
    if not native(logits):
        return TF.cross_entropy(logits, labels, label_smoothing=label_smoothing)
    if logits.dtype not in (BF16, F32) or not logits.is_contiguous():
        logits = logits.contiguous()
        if logits.dtype not in (BF16, F32):
            logits = logits.float()
    labels = labels.contiguous().long()
    return _XentFn.apply(logits, labels, float(label_smoothing))


# ------------------------------------------------------------------------------------------
# Linear classifier + softmax cross-entropy in pieces of the vocabulary (csrc/linear_xent.hip): the
# logits are never in memory as a whole, forward or backward.
# ------------------------------------------------------------------------------------------
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _counted(labels, V, ignore_index):
    return (labels != ignore_index) & (labels >= 0) & (labels < V)


def _linear_xent_plain(x, weight, labels, bias, smoothing, ignore_index, reduction):
    """The same loss in torch operations: the rows that do not count are left out before the product."""
    V = weight.shape[0]
    keep = _counted(labels, V, ignore_index)
    wide = torch.float64 if x.dtype == torch.float64 else F32
    logits = TF.linear(x[keep].to(wide), weight.to(wide), bias.to(wide) if bias is not None else None)
    rows = TF.cross_entropy(logits, labels[keep], reduction="none", label_smoothing=smoothing)
    if reduction == "none":
        return torch.zeros(labels.shape, dtype=wide, device=x.device).masked_scatter(keep, rows)
    return rows.sum() / max(rows.numel(), 1) if reduction == "mean" else rows.sum()


def _is_operand(t, D, Dp):
    return (t.dtype == BF16 and D == Dp and t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0
            and D <= t.stride(0) <= 1 << 22)


def _operands(x, weight, D, Dp):
    """x and weight (None: not wanted) as bf16 operands of the products: rows of Dp columns (zeros behind D) on
    16 bytes. A tensor that is one already itself, the others packed in one launch."""
    out, args = [], []
    for t in (x, weight):
        if t is None or _is_operand(t, D, Dp):
            out.append(t)
            args += (0, 0, 0, 0, 0)
            continue
        if t.stride(1) != 1 or t.stride(0) < D:
            t = t.contiguous()
        k = t.new_empty((t.shape[0], Dp), dtype=BF16)
        out.append(k)
        args += (ptr(t), int(t.dtype == BF16), max(t.stride(0), D), t.shape[0], ptr(k))
    if any(args):
        lib().pack_rows(*args, D, Dp, stream_handle())
    return out


def _cached_weight(weight):
    """fp32 parameters keep their bf16 operand from step to step (ops/wcache.py). A captured pass that is not
    part of a captured training step lays out its own, in every replay."""
    return (weight.dtype == F32 and isinstance(weight, torch.nn.Parameter) and weight.is_contiguous()
            and not wcache.outdated_in_replays())


def _operand(weight, Dp):
    from .conv import _prep_weight

    V, D = weight.shape
    return _prep_weight(weight.view(V, D, 1, 1), 1, Dp, mode=0, param=weight).view(V, Dp)


def _linear_xent_args(xk, wk, b, labels, V, Dp, D, ignore_index, smoothing, reduction):
    N = xk.shape[0]
    return (ptr(xk), xk.stride(0) if N > 1 else Dp, ptr(wk), wk.stride(0) if V > 1 else Dp, ptr(b), ptr(labels), N, V, Dp, D,
            ignore_index, smoothing, reduction)


def _linear_xent_forward(x, weight, bias, labels, smoothing, ignore_index, reduction, train):
    """(loss, what backward needs beside x and weight)."""
    N, D = x.shape
    V, dev = weight.shape[0], x.device
    Dp = (D + 63) // 64 * 64
    cached = _cached_weight(weight)
    xk, wk = _operands(x, None if cached else weight, D, Dp)
    if cached:
        wk = _operand(weight, Dp)
    b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    args = _linear_xent_args(xk, wk, b, labels, V, Dp, D, ignore_index, smoothing, reduction)
    need = lib().linear_xent_fwd_bytes(*args)
    if need < 0:
        raise ValueError(f"linear_cross_entropy: {N} rows against {V} classes are more than a call takes")
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    # per row (largest logit, log2 of the sum above it); behind them (sum of the losses, rows that count)
    stats = torch.empty(2 * N + 2, dtype=F32, device=dev)
    loss = torch.empty(() if reduction else N, dtype=F32, device=dev)
    at = stats.data_ptr()
    if reduction:
        lib().linear_xent_fwd(*args, ptr(ws), at if train else 0, 0, at + 8 * N, ptr(loss), stream_handle())
    else:
        lib().linear_xent_fwd(*args, ptr(ws), at if train else 0, ptr(loss), 0, 0, stream_handle())
    return loss, (labels, xk, None if cached else wk, b, stats)


class _LinearXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, labels, smoothing, ignore_index, reduction, leaf):  # leaf: the caller's x
        with on_device(x):
            track_leaves(ctx, *leaf, weight, bias)
            loss, saved = _linear_xent_forward(x, weight, bias, labels, smoothing, ignore_index, reduction, True)
        ctx.cfg = (smoothing, ignore_index, reduction)
        # backward reads the parameter's own operand and the bias again, unless the forward pass made copies
        ctx.seen = (updates_seen(weight if saved[2] is None else None), updates_seen(bias if saved[3] is bias else None))
        ctx.save_for_backward(x, weight, bias, *saved)
        return loss

    @staticmethod
    def backward(ctx, go):
        return first_derivative_only("linear_cross_entropy", _linear_xent_backward, ctx, go)


def _linear_xent_backward(ctx, go, sinks):
    x, weight, bias, labels, xk, wk, b, stats = ctx.saved_tensors
    smoothing, ignore_index, reduction = ctx.cfg
    refuse_updated("linear_cross_entropy", "weight", weight, ctx.seen[0])
    refuse_updated("linear_cross_entropy", "bias", bias, ctx.seen[1])
    N, D = x.shape
    V, Dp = weight.shape[0], (D + 63) // 64 * 64
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    sw = accumulation_sink(ctx, 1, weight) if need_w and sinks else None
    sb = accumulation_sink(ctx, 2, bias) if need_b and sinks else None
    dx = x.new_empty((N, D)) if need_x else None
    dw = sw if sw is not None else weight.new_empty((V, D)) if need_w else None
    db = sb if sb is not None else bias.new_empty(V) if need_b else None
    if go.dtype != F32 or not go.is_contiguous():
        go = go.to(F32).contiguous()
    # (the engine runs a node on the device and stream of its forward pass)
    if wk is None:  # the parameter's operand
        wk = _operand(weight, Dp)
    args = _linear_xent_args(xk, wk, b, labels, V, Dp, D, ignore_index, smoothing, reduction)
    ws = x.new_empty(lib().linear_xent_bwd_bytes(*args, int(need_x), int(need_w), int(need_b)), dtype=torch.uint8)
    at = stats.data_ptr()
    lib().linear_xent_bwd(*args, ptr(go), at + 8 * N, ptr(ws), at, ptr(dx), ptr(dw),
                          int(weight.dtype == F32), int(sw is not None), ptr(db), int(sb is not None), stream_handle())
    return dx, None if sw is not None else dw, None if sb is not None else db, None, None, None, None, None


_apply_linear_xent = fast_apply(_LinearXentFn)


def linear_cross_entropy(x, weight, labels, bias=None, label_smoothing=0.0, ignore_index=-100, reduction="mean"):
    """Cross-entropy of ``softmax(x @ weight.T + bias)`` against ``labels``, with its gradients for x,
    weight and bias, in pieces of the vocabulary: the logits are never kept (csrc/linear_xent.hip).

    x (..., D) bf16 (fp32 is rounded to it, as ``linear`` does); weight (V, D) bf16, or the fp32
    parameter, used through its bf16 operand; bias (V,) fp32 or None; labels (...) integers. Rows whose
    label is ``ignore_index`` or lies outside [0, V) take no part: their loss and gradient are zero
    whatever x holds there. ``reduction`` is "mean" over the rows that count (0 if none does), "sum",
    or "none" (labels' shape). Products are summed in fp32, the loss and bias gradient are fp32, the
    gradient of the logits is rounded to bf16 for the two products behind it; the weight's gradient
    has the weight's type and goes straight into a live ``.grad`` buffer. At most 2^22 rows, 2^30 classes
    and 2^38 logits. As for ``linear``, the operand of a parameter follows its in-place changes and the fused
    optimizers; what is written through ``.data`` shows from the next step on (or behind ``ops.wcache.clear()``)."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"linear_cross_entropy: x {tuple(x.shape)} does not match weight {tuple(weight.shape)} (V, D)")
    if labels.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: labels {tuple(labels.shape)} do not match x {tuple(x.shape)}")
    if labels.dtype not in (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8):
        raise TypeError(f"linear_cross_entropy: labels must be integers, got {labels.dtype}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"linear_cross_entropy: bias has shape {tuple(bias.shape)}, expected ({weight.shape[0]},)")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"linear_cross_entropy: label_smoothing must lie in [0, 1], got {label_smoothing}")
    same_device("linear_cross_entropy", x, weight, labels, bias)
    D = x.shape[-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, D)
    flat = labels if labels.dim() == 1 else labels.reshape(-1)
    if flat.dtype != torch.int64:
        flat = flat.long()
    for name, t, kinds in (("x", x, (BF16, F32)), ("weight", weight, (BF16, F32)), ("bias", bias, (F32,))):
        if t is not None and t.dtype not in kinds and native(x):
            raise TypeError(f"linear_cross_entropy: {name} must be {' or '.join(str(k)[6:] for k in kinds)}, got {t.dtype}")
    if not native(x) or not x2.shape[0]:
        loss = _linear_xent_plain(x2, weight, flat, bias, float(label_smoothing), int(ignore_index), reduction)
        return loss.reshape(labels.shape) if reduction == "none" else loss
    if x2.shape[0] > int(lib().XENT_MAX_ROWS):
        raise ValueError(f"linear_cross_entropy: {x2.shape[0]} rows, at most {int(lib().XENT_MAX_ROWS)} in a call")
    V = weight.shape[0]
    if V > int(lib().XENT_MAX_CLASSES) or (V // 32 + 1) * (x2.shape[0] // 32 + 1) >= 1 << 31:
        raise ValueError(f"linear_cross_entropy: {x2.shape[0]} rows against {V} classes are more than a call takes")
    if D > 1 << 22:
        raise ValueError(f"linear_cross_entropy: rows of {D} values, at most {1 << 22}")
    code = _REDUCTIONS[reduction]
    if x2.dtype != BF16:
        x2 = x2.to(BF16)
    args = (x2, weight, bias, flat if flat.is_contiguous() else flat.contiguous(), float(label_smoothing), int(ignore_index), code)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x2, weight, bias))) or observed():
        loss = _apply_linear_xent(*args, (x,))
    else:
        with on_device(x):
            loss = _linear_xent_forward(x2, weight, bias, *args[3:], False)[0]
    return loss if code else loss.reshape(labels.shape)


# ------------------------------------------------------------------------------------------
# Pointwise losses (csrc/losses.hip): one pass computes the sum, the backward launch writes the
# gradient scaled by the upstream gradient read from device memory (no host synchronisation).
# ------------------------------------------------------------------------------------------
_KINDS = {"wmse": 0, "mse": 1, "l1": 2, "bce_logits": 3, "focal": 4}


def _rows(x):
    """(rows, C, ld) of the physical layout of ``x`` (NHWC 4-D or contiguous)."""
    from .common import is_nhwc, ld_of

    if x.dim() == 4 and is_nhwc(x):
        N, C, H, W = x.shape
        return N * H * W, C, ld_of(x)
    return x.numel(), 1, 1


def _native_pred(x):
    from .common import is_nhwc

    if x.dim() == 4 and is_nhwc(x):
        return x
    if x.dtype in (BF16, F32) and x.is_contiguous():
        return x
    if x.dim() == 4:
        return x.to(BF16).contiguous(memory_format=torch.channels_last)
    return x.contiguous()


def _match_target(t, pred):
    if pred.dim() == 4 and pred.stride(1) == 1 and pred.shape[1] > 1:
        t = t.contiguous(memory_format=torch.channels_last)
    else:
        t = t.contiguous()
    if t.dtype not in (BF16, F32):
        t = t.float()
    return t, (1 if t.dtype == BF16 else 0)


class _PWLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, target, tval, kind, a, b, norm, weight=None):
        rows, C, ld = _rows(pred)
        dev = pred.device
        sums = torch.zeros(2, dtype=F32, device=dev)
        if target is not None:
            target, ttype = _match_target(target, pred)
        else:
            ttype = 2
        if weight is not None:
            weight = _match_target(weight.float(), pred)[0]
        lib().pw_loss(kind, ptr(pred), int(pred.dtype == BF16), ptr(target), ttype, float(tval), ptr(weight), rows, C,
                      ld, C, a, b, ptr(sums), 0, 0, 1.0, stream_handle())
        if kind == _KINDS["focal"]:
            scale = 1.0 / sums[1].clamp(min=1.0)
        else:
            scale = torch.full((), norm, dtype=F32, device=dev)
        ctx.save_for_backward(pred, target, scale, weight)
        ctx.cfg = (tval, kind, a, b, ttype)
        return sums[0] * scale

    @staticmethod
    def backward(ctx, gout):
        pred, target, scale, weight = ctx.saved_tensors
        tval, kind, a, b, ttype = ctx.cfg
        rows, C, ld = _rows(pred)
        gs = (gout.float() * scale).reshape(1).contiguous()
        if pred.dim() == 4 and ld != pred.shape[1]:
            from .common import empty_nhwc

            grad = empty_nhwc(*pred.shape, pred.device)
        else:
            grad = torch.empty_like(pred)
        lib().pw_loss(kind, ptr(pred), int(pred.dtype == BF16), ptr(target), ttype, float(tval), ptr(weight), rows, C,
                      ld, C, a, b, 0, ptr(grad), ptr(gs), 1.0, stream_handle())
        return grad, None, None, None, None, None, None, None


def _pw(pred, target, kind, a=0.0, b=0.0, reduction="mean", weight=None, norm=None):
    if isinstance(target, (int, float)):
        tval, target_t = float(target), None
    else:
        tval, target_t = 0.0, target
    if weight is not None and target_t is None:
        target_t = torch.full(pred.shape, tval, dtype=F32, device=pred.device)
    pred = _native_pred(pred)
    if norm is None:
        norm = 1.0 / pred.numel() if reduction == "mean" else 1.0
    return _PWLossFn.apply(pred, target_t, tval, _KINDS[kind], float(a), float(b), norm, weight)


def _full_like(t, v):
    return torch.full_like(t, v) if isinstance(v, (int, float)) else v


def heatmap_mse(pred, target, fg_weight=81.0):
    """mean((t - p)^2 * (1 + fg_weight [t > 0])) -- the Hourglass loss of one stack
    (R/Hourglass/tensorflow/train.py:65-76; the trainer divides by the global batch)."""
    if not native(pred):
        w = (target > 0).float() * fg_weight + 1
        return ((target - pred.float()) ** 2 * w).mean()
    return _pw(pred, target, "wmse", a=fg_weight)


def mse_loss(pred, target, reduction="mean"):
    """MSE against a tensor or a constant label (LSGAN, R/CycleGAN/tensorflow/train.py:53-62)."""
    if not native(pred):
        d = (pred.float() - _full_like(pred.float(), target)) ** 2
        return d.mean() if reduction == "mean" else d.sum()
    return _pw(pred, target, "mse", reduction=reduction)


def l1_loss(pred, target, reduction="mean"):
    if not native(pred):
        d = (pred.float() - _full_like(pred.float(), target).float()).abs()
        return d.mean() if reduction == "mean" else d.sum()
    return _pw(pred, target, "l1", reduction=reduction)


def bce_with_logits(logits, target, reduction="mean"):
    """tf.keras.losses.BinaryCrossentropy(from_logits=True) (R/DCGAN/tensorflow/main.py:42-53)."""
    if not native(logits):
        return TF.binary_cross_entropy_with_logits(logits.float(), _full_like(logits.float(), target).float(),
                                                   reduction=reduction)
    return _pw(logits, target, "bce_logits", reduction=reduction)


def focal_loss(logits, target, alpha=2.0, beta=4.0):
    """CenterNet penalty-reduced pixel-wise focal loss on sigmoid(logits), normalised by the number
    of positive (t == 1) locations."""
    if not native(logits):
        p = torch.sigmoid(logits.float()).clamp(1e-4, 1 - 1e-4)
        t = target.float()
        pos = t.ge(1).float()
        lp = -((1 - p) ** alpha) * torch.log(p) * pos
        ln = -((1 - t) ** beta) * p ** alpha * torch.log(1 - p) * (1 - pos)
        return (lp.sum() + ln.sum()) / pos.sum().clamp(min=1)
    return _pw(logits, target, "focal", a=alpha, b=beta, reduction="sum")


def masked_l1(pred, target, mask, num=None):
    """sum(|p - t| * mask) / max(num, 1) -- CenterNet size / offset regression at object centres
    (``mask`` in the target's shape; ``num`` a host count, default ``mask.sum()`` synced)."""
    n = float(max(1.0, float(mask.sum()) if num is None else num))
    if not native(pred):
        return ((pred.float() - target.float()).abs() * mask.float()).sum() / n
    return _pw(pred, target, "l1", weight=mask, norm=1.0 / n)
