"""Class loss of a rendered feature map: ``class_cross_entropy(features, weight, labels, bias)``.

The softmax cross entropy of every pixel's (or row's) label through a linear
classifier ``z = weight @ f + bias``, as identity and language fields are
trained: the scene's per-Gaussian features are rendered to a (C,H,W) map and
each pixel is classified.  The V logits of a pixel are never stored (at
1920x1080 and 256 classes they would be 2.1 GB): forward streams the classes
past the pixels with a running maximum and sum, backward recomputes them tile
by tile and accumulates the gradients of the map, the classifier and its bias.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib, _pipeline

__all__ = ["class_cross_entropy"]

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
MAX_CHANNELS = 256
MAX_CHANNELS_FP32 = 128
TILE = 128


def _validate(features, weight, labels, bias, ignore_index, reduction, train) -> None:
    if not all(isinstance(t, torch.Tensor) for t in (features, weight, labels)):
        raise ValueError("features, weight and labels must be torch.Tensor instances")
    if features.ndim not in (2, 3, 4):
        raise ValueError("features must have shape (N, C), (C, H, W) or (B, C, H, W)")
    channels = features.shape[0] if features.ndim == 3 else features.shape[1]
    shape = {2: features.shape[:1], 3: features.shape[1:],
             4: features.shape[:1] + features.shape[2:]}[features.ndim]
    if labels.shape != shape:
        raise ValueError(f"labels must have shape {tuple(shape)}, got {tuple(labels.shape)}")
    if weight.ndim != 2 or weight.shape[1] != channels or weight.shape[0] < 1:
        raise ValueError(f"weight must have shape (V, {channels}) with V >= 1, got {tuple(weight.shape)}")
    if features.dtype not in _lib.DTYPES or weight.dtype != features.dtype:
        raise ValueError("features and weight must share one dtype of float32, bfloat16 and float16, "
                         f"got {features.dtype} and {weight.dtype}")
    if labels.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"labels must have dtype int32 or int64, got {labels.dtype}")
    limit = MAX_CHANNELS_FP32 if features.dtype == torch.float32 else MAX_CHANNELS
    if not 1 <= channels <= limit:
        raise ValueError(f"{features.dtype} features must have 1 to {limit} channels, got {channels}")
    if labels.numel() >= (1 << 31) - TILE or weight.shape[0] >= (1 << 31) - TILE:
        raise ValueError("rows and classes must be fewer than 2**31 - 128")
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.shape != weight.shape[:1] or bias.dtype != torch.float32:
            raise ValueError(f"bias must be a float32 tensor of shape ({weight.shape[0]},)")
    if not features.is_cuda or any(t is not None and t.device != features.device for t in (weight, labels, bias)):
        raise ValueError("features, weight, labels and bias must be on the same CUDA device")
    if not isinstance(ignore_index, int) or isinstance(ignore_index, bool):
        raise ValueError("ignore_index must be an int")
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError("ignore_index must fit 64 bits")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    if not isinstance(train, bool):
        raise ValueError("train must be a bool")


def _rows(features):
    """(B, S, C, strides of b, c and s): rows n = b * S + s of a map or a matrix.  A map whose pixels have
    no single stride is made contiguous first."""
    x = features
    if x.ndim == 2:
        x = x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()
        # stride_c = 1 marks rows of channels: the gradient is written (N, C)
        return x, 1, x.shape[0], x.shape[1], (0, 1, x.stride(0))
    B, C, H, W = (1, *x.shape) if x.ndim == 3 else x.shape
    sb, sc, sh, sw = (0, *x.stride()) if x.ndim == 3 else x.stride()
    if (H > 1 and sh != W * sw) or (sc == 1 and C > 1):
        x = x.contiguous()
        sb, sc, sw = C * H * W, H * W, 1
    return x, B, H * W, C, (sb, max(sc, 2) if C == 1 else sc, sw)


def _forward(features, weight, labels, bias, ignore_index, reduction, train=True):
    """``(loss, args, kept, bytes of the backward workspace)``: the argument block with its sizes, and the
    buffer that backward reads."""
    x, B, S, C, (sb, sc, ss) = _rows(features)
    dev = x.device
    N = B * S
    w = weight.contiguous()
    b = bias.contiguous() if bias is not None else None
    y = labels.contiguous()
    a = _lib.ClassLossArgs(B, S, w.shape[0], C, _lib.DTYPES[x.dtype], _REDUCTIONS[reduction],
                           labels.dtype == torch.int64, train, sb, sc, ss, ignore_index,
                           x.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(), y.data_ptr())
    sizes = _SIZES()
    _lib.call("gsb_class_loss_sizes", a, sizes)
    # torch's allocations are 512-byte aligned
    kept = torch.empty(sizes[0], dtype=torch.uint8, device=dev)
    ws = torch.empty(sizes[1], dtype=torch.uint8, device=dev)
    # one element at least: an empty tensor has no address
    loss = torch.empty(max(N, 1) if reduction == "none" else 1, dtype=torch.float32, device=dev)
    a.loss, a.kept, a.workspace, a.workspace_bytes = loss.data_ptr(), kept.data_ptr(), ws.data_ptr(), sizes[1]
    a.error_word = _pipeline.sticky_error_word(dev).data_ptr()
    with _pipeline._stage_timer("class_loss_fwd", {"rows": N}):
        _lib.call_on(dev, "gsb_class_loss_fwd", a)
    loss = loss[:N].view(labels.shape) if reduction == "none" else loss.view(())
    return loss, a, kept, sizes[2]


_SIZES = ctypes.c_size_t * 3


def _backward(args, kept, ws_bytes, upstream, features_shape, dtype, want_features, want_weight, want_bias):
    dev = kept.device
    a = _lib.ClassLossArgs.from_buffer_copy(args)
    a.features = a.weight = a.bias = a.labels = a.loss = None  # not kept, not read
    up = upstream if upstream.dtype == torch.float32 else upstream.float()
    up = up.contiguous()
    gx = torch.empty(features_shape, dtype=dtype, device=dev) if want_features else None
    gw = torch.empty((a.V, a.C), dtype=dtype, device=dev) if want_weight else None
    gb = torch.empty(a.V, dtype=torch.float32, device=dev) if want_bias else None
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    a.kept, a.workspace, a.workspace_bytes = kept.data_ptr(), ws.data_ptr(), ws_bytes
    a.upstream = up.data_ptr()
    if want_features:
        a.grad_features = gx.data_ptr()
    if want_weight:
        a.grad_weight = gw.data_ptr()
    if want_bias:
        a.grad_bias = gb.data_ptr()
    with _pipeline._stage_timer("class_loss_bwd", {"rows": a.B * a.S}):
        _lib.call_on(dev, "gsb_class_loss_bwd", a)
    return gx, gw, gb


class _ClassCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, weight, labels, bias, ignore_index, reduction):
        loss, ctx.args, kept, ctx.ws_bytes = _forward(features, weight, labels, bias, ignore_index, reduction)
        ctx.shape, ctx.dtype = features.shape, features.dtype
        ctx.save_for_backward(kept)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        want = ctx.needs_input_grad
        if not (want[0] or want[1] or want[3]):
            return (None,) * 6
        kept, = ctx.saved_tensors
        gx, gw, gb = _backward(ctx.args, kept, ctx.ws_bytes, grad, ctx.shape, ctx.dtype, want[0], want[1], want[3])
        return gx, gw, None, gb, None, None


def class_cross_entropy(features, weight, labels, bias=None, ignore_index=-100, reduction="mean", train=True):
    """Softmax cross entropy of ``labels`` under the logits ``weight @ f + bias`` of every pixel or row ``f``.

    ``features`` is a map (C, H, W) or (B, C, H, W), or rows (N, C); ``labels`` (int32 or int64) has its shape
    without C.  ``weight`` (V, C) shares the features' type: float32 with up to 128 channels, bfloat16 or float16
    with up to 256.  ``bias`` (V,) is float32.  Logits, softmax and sums are float32 and gradients are rounded
    once to their input's type; for 16-bit inputs the softmax's probabilities are rounded to 16 bits of precision
    before the gradients' products (to bfloat16's 8 for bfloat16 inputs of more than 8 channels and 128 classes).

    Returns a float32 scalar ("mean" over the rows that count, "sum") or the rows' losses in ``labels``' shape
    ("none").  Rows labelled ``ignore_index`` have loss 0 and no gradient, whatever their features hold; with no
    row left the mean is 0.  Labels outside [0, V) count as ignored and are reported by the device error word (a
    ``RuntimeError`` from ``raise_device_errors``, or from the next rasterizer call, which reads it too).  A class
    whose bias is -inf takes no part (its weight row is not read); a row labelled with it has the loss +inf and no
    gradient.  Finite biases beyond 2e38 in magnitude count as 2e38.

    With ``train`` the loss is differentiable in ``features``, ``weight`` and ``bias``; the call then keeps a
    packed copy of the features and the classifier instead of the tensors themselves.  Where no gradient can be
    asked for (none of them requires one, or gradients are off) the call is a forward alone, as with ``train=False``.
    """
    _validate(features, weight, labels, bias, ignore_index, reduction, train)
    if not (train and torch.is_grad_enabled()
            and (features.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))):
        with torch.no_grad():
            return _forward(features, weight, labels, bias, ignore_index, reduction, False)[0]
    return _ClassCrossEntropy.apply(features, weight, labels, bias, ignore_index, reduction)
