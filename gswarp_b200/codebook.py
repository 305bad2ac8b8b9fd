"""Shared attribute rows: ``codebook_lookup(table, codes, scale)`` and its gradients.

A compressed scene keeps one code per Gaussian and a codebook of attribute
rows (SH rows, DC colours, feature rows).  The lookup expands the rows the
rasterizer takes (``dc``, ``shs``, ``colors_precomp``); backward sums the
rows' gradients by sorted code, without atomics, so it gives the same bits on
every call.  ``scale`` is one factor, or a gain per Gaussian (shape-gain
codebooks), which gets a gradient too.
"""

from __future__ import annotations

import math
from numbers import Real

import torch

from . import _lib, _pipeline

__all__ = ["codebook_lookup"]

_INDEX_TYPES = (torch.int32, torch.int64)
MAX_COLS = 1 << 22
MAX_ROWS = (1 << 31) - 4096


def _validate(table, codes, scale) -> None:
    if not (isinstance(table, torch.Tensor) and isinstance(codes, torch.Tensor)):
        raise ValueError("table and codes must be torch.Tensor instances")
    shape = table.shape
    if len(shape) < 2:
        raise ValueError(f"table must have shape (K, ...) with at least two dimensions, got {tuple(shape)}")
    if table.dtype not in _lib.DTYPES:
        raise ValueError(f"table must have dtype float32, bfloat16 or float16, got {table.dtype}")
    if codes.dtype not in _INDEX_TYPES:
        raise ValueError(f"codes must have dtype int32 or int64, got {codes.dtype}")
    device = table.device
    if not table.is_cuda or codes.device != device:
        raise ValueError("table and codes must be on the same CUDA device")
    row = shape[1] if len(shape) == 2 else math.prod(shape[1:])
    if not 1 <= row <= MAX_COLS:
        raise ValueError(f"table rows must have 1 to {MAX_COLS} elements, got {row}")
    if shape[0] >= (1 << 31) - 1 or codes.numel() >= MAX_ROWS:
        raise ValueError("table and codes must have fewer than 2**31 - 4096 rows")
    if type(scale) is float:
        return
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.shape != codes.shape or scale.device != device:
            raise ValueError("a scale tensor must be float32 with the shape and device of codes")
    elif not isinstance(scale, Real) or isinstance(scale, bool):
        raise ValueError("scale must be a number or a float32 tensor")


# The small calls' time is the host's (10,000 x 3 in training: 10 us of kernels, 75 of a pass), and half of that is
# autograd's; what runs once per call below is kept short.


def _call(device, stage, name, a) -> None:
    with _pipeline._stage_timer(stage, {"rows": a.P}):
        _lib.call_on(device, name, a)


def _forward(table, codes, scale, gain, out):
    """The rows, and the argument block, of contiguous tensors."""
    dev, dtype, shape = table.device, table.dtype, table.shape
    P = codes.numel()
    if len(shape) == 2:
        K, D = shape
    else:
        K, D = shape[0], math.prod(shape[1:])
    if out is None:
        if len(shape) == 2 and codes.ndim == 1:
            out = torch.empty_strided((P, D), (D, 1), dtype=dtype, device=dev)  # the quickest of torch's ways
        else:
            out = torch.empty(codes.shape + shape[1:], dtype=dtype, device=dev)
    a = _lib.CodebookArgs(P, K, D, _lib.DTYPES[dtype], codes.dtype is torch.int64, scale, table.data_ptr(),
                          codes.data_ptr(), None if gain is None else gain.data_ptr(), out.data_ptr(), None, None, None,
                          _pipeline.sticky_error_word(dev).data_ptr())
    if _pipeline.TIMING_ENABLED:
        _call(dev, "codebook_fwd", "gsb_codebook_fwd", a)
    else:
        _lib.call_on(dev, "gsb_codebook_fwd", a)
    return out, a


def lookup_forward(table: torch.Tensor, codes: torch.Tensor, scale: float = 1.0,
                   gain: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * gain * table[codes]`` of contiguous tensors, into ``out`` if given."""
    return _forward(table, codes, scale, gain, out)[0]


def _backward(a, shape, codes, gain, grad_out, want_table, want_gain, out):
    """Gradients for the argument block ``a``, whose table, codes and gains are set."""
    dev = grad_out.device
    a.grad_out = grad_out.data_ptr()
    grad_table = grad_gain = None
    if want_table:
        if out is not None:
            grad_table = out
        elif len(shape) == 2:
            grad_table = torch.empty_strided(shape, (shape[1], 1), dtype=grad_out.dtype, device=dev)
        else:
            grad_table = torch.empty(shape, dtype=grad_out.dtype, device=dev)
        a.grad_table = grad_table.data_ptr()
        n = _lib.load().gsb_codebook_bwd_workspace_bytes(a.P, a.K, a.D)
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
    if want_gain:
        grad_gain = torch.empty(codes.shape, dtype=torch.float32, device=dev)
        a.grad_gain = grad_gain.data_ptr()
        if gain is None:
            a.gain = a.grad_gain  # there have to be gains, but their own gradient does not read them
    if _pipeline.TIMING_ENABLED:
        _call(dev, "codebook_bwd", "gsb_codebook_bwd", a)
    else:
        _lib.call_on(dev, "gsb_codebook_bwd", a)
    return grad_table, grad_gain


def lookup_backward(shape, dtype, table: torch.Tensor | None, codes: torch.Tensor, scale: float,
                    gain: torch.Tensor | None, grad_out: torch.Tensor, want_table: bool = True,
                    want_gain: bool = False, out: torch.Tensor | None = None):
    """``(grad_table, grad_gain)`` of contiguous tensors, for a table of ``shape`` and ``dtype``; ``grad_table`` into
    ``out`` if given.  The table is read only for the gains' gradient, the gains only for the table's."""
    a = _lib.CodebookArgs(codes.numel(), shape[0], math.prod(shape[1:]), _lib.DTYPES[dtype], codes.dtype is torch.int64,
                          scale, None if table is None else table.data_ptr(), codes.data_ptr(),
                          None if gain is None else gain.data_ptr())
    a.error_word = _pipeline.sticky_error_word(grad_out.device).data_ptr()
    return _backward(a, shape, codes, gain, grad_out, want_table, want_gain, out)


class _CodebookLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, codes, scale, gain):
        t = table.contiguous()
        c = codes.contiguous()
        g = gain.contiguous() if gain is not None else None
        out, ctx.args = _forward(t, c, scale, g, None)
        ctx.shape = table.shape
        # what no gradient reads may change before backward: the table's reads the gains, the gains' the table
        want_table, _, _, want_gain = ctx.needs_input_grad
        ctx.save_for_backward(c, g if want_table else None, t if want_gain else None)
        return out

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():  # a graph of this pass is asked for: a second derivative is refused
            return _once(ctx, grad)
        want_table, _, _, want_gain = ctx.needs_input_grad
        if not (want_table or want_gain):
            return None, None, None, None
        a = _lib.CodebookArgs.from_buffer_copy(ctx.args)
        c, g, t = ctx.saved_tensors
        a.codes = c.data_ptr()
        a.gain = None if g is None else g.data_ptr()
        a.table = None if t is None else t.data_ptr()
        grad_table, grad_gain = _backward(a, ctx.shape, c, g, grad.contiguous(), want_table, want_gain, None)
        return grad_table, None, None, grad_gain


_once = torch.autograd.function.once_differentiable(_CodebookLookup.backward)

# Function.apply's part in Python is there for functorch's transforms, which it refuses for this class.
_apply = super(torch.autograd.Function, _CodebookLookup).apply


def codebook_lookup(table, codes, scale=1.0):
    """``scale * table[codes]``: rows of a codebook ``(K, ...)`` (float32, bfloat16 or float16) for ``codes`` of
    any shape (int32 or int64), of shape ``codes.shape + table.shape[1:]`` and the table's type.

    ``scale`` is a number, or a float32 tensor of ``codes``' shape (one gain per row).  Products are taken in
    float32 and rounded once.  Code -1 gives a zero row and no gradient; any other code outside ``[0, K)`` does
    the same and is reported by the device error word (a ``RuntimeError`` from ``raise_device_errors``, or from the
    next rasterizer call, which reads it too).
    Differentiable in ``table`` and in a tensor ``scale``.
    """
    _validate(table, codes, scale)
    gain = None
    if isinstance(scale, torch.Tensor):
        gain, scale = scale, 1.0
    else:
        scale = float(scale)
    if not (torch.is_grad_enabled() and (table.requires_grad or (gain is not None and gain.requires_grad))):
        return lookup_forward(table.contiguous(), codes.contiguous(), scale,
                              None if gain is None else gain.contiguous())
    if torch._C._are_functorch_transforms_active():
        return _CodebookLookup.apply(table, codes, scale, gain)
    return _apply(table, codes, scale, gain)
