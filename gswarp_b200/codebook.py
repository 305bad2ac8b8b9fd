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


def _validate(table, codes, scale) -> None:
    if not isinstance(table, torch.Tensor) or not isinstance(codes, torch.Tensor):
        raise ValueError("table and codes must be torch.Tensor instances")
    if table.ndim < 2:
        raise ValueError(f"table must have shape (K, ...) with at least two dimensions, got {tuple(table.shape)}")
    if table.dtype not in _lib.DTYPES:
        raise ValueError(f"table must have dtype float32, bfloat16 or float16, got {table.dtype}")
    if codes.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"codes must have dtype int32 or int64, got {codes.dtype}")
    if not table.is_cuda or codes.device != table.device:
        raise ValueError("table and codes must be on the same CUDA device")
    row = math.prod(table.shape[1:])
    if row < 1 or row > 1 << 22:
        raise ValueError(f"table rows must have 1 to {1 << 22} elements, got {row}")
    if table.shape[0] >= (1 << 31) - 1 or codes.numel() >= (1 << 31) - 4096:
        raise ValueError("table and codes must have fewer than 2**31 - 4096 rows")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.shape != codes.shape or scale.device != codes.device:
            raise ValueError("a scale tensor must be float32 with the shape and device of codes")
    elif not isinstance(scale, Real) or isinstance(scale, bool):
        raise ValueError("scale must be a number or a float32 tensor")


def _args(shape, dtype, table, codes, scale, gain, device) -> _lib.CodebookArgs:
    a = _lib.CodebookArgs(codes.numel(), shape[0], math.prod(shape[1:]), _lib.DTYPES[dtype],
                          codes.dtype == torch.int64, scale, None if table is None else table.data_ptr(),
                          codes.data_ptr(), None if gain is None else gain.data_ptr())
    a.error_word = _pipeline.sticky_error_word(device).data_ptr()
    return a


def lookup_forward(table: torch.Tensor, codes: torch.Tensor, scale: float = 1.0,
                   gain: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * gain * table[codes]`` of contiguous tensors, into ``out`` if given."""
    dev = table.device
    if out is None:
        out = torch.empty(codes.shape + table.shape[1:], dtype=table.dtype, device=dev)
    a = _args(table.shape, table.dtype, table, codes, scale, gain, dev)
    a.out = out.data_ptr()
    with _pipeline._stage_timer("codebook_fwd", {"rows": a.P, "kernels": 1}):
        _lib.call_on(dev, "gsb_codebook_fwd", a)
    return out


def lookup_backward(shape, dtype, table: torch.Tensor | None, codes: torch.Tensor, scale: float,
                    gain: torch.Tensor | None, grad_out: torch.Tensor, want_table: bool = True,
                    want_gain: bool = False, out: torch.Tensor | None = None):
    """``(grad_table, grad_gain)`` of contiguous tensors, for a table of ``shape`` and ``dtype``; ``grad_table`` into
    ``out`` if given.  The table is read only for the gains' gradient, the gains only for the table's."""
    dev = grad_out.device
    a = _args(shape, dtype, table, codes, scale, gain, dev)
    a.grad_out = grad_out.data_ptr()
    grad_table = grad_gain = None
    if want_table:
        grad_table = torch.empty(shape, dtype=dtype, device=dev) if out is None else out
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
    with _pipeline._stage_timer("codebook_bwd", {"rows": a.P}):
        _lib.call_on(dev, "gsb_codebook_bwd", a)
    return grad_table, grad_gain


class _CodebookLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, codes, scale, gain):
        t = table.contiguous()
        c = codes.contiguous()
        ctx.scale, ctx.shape, ctx.dtype = scale, table.shape, table.dtype
        g = gain.contiguous() if gain is not None else None
        # what no gradient reads may change before backward: the table's reads the gains, the gains' the table
        want_table, _, _, want_gain = ctx.needs_input_grad
        ctx.save_for_backward(c, g if want_table else None, t if want_gain else None)
        return lookup_forward(t, c, scale, g)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        want_table, _, _, want_gain = ctx.needs_input_grad
        if not (want_table or want_gain):
            return None, None, None, None
        c, g, t = ctx.saved_tensors
        grad_table, grad_gain = lookup_backward(ctx.shape, ctx.dtype, t, c, ctx.scale, g, grad.contiguous(), want_table,
                                                want_gain)
        return grad_table, None, None, grad_gain


def codebook_lookup(table, codes, scale=1.0):
    """``scale * table[codes]``: rows of a codebook ``(K, ...)`` (float32, bfloat16 or float16) for ``codes`` of
    any shape (int32 or int64), of shape ``codes.shape + table.shape[1:]`` and the table's type.

    ``scale`` is a number, or a float32 tensor of ``codes``' shape (one gain per row).  Products are taken in
    float32 and rounded once.  Code -1 gives a zero row and no gradient; any other code outside ``[0, K)`` does
    the same and is reported by the device error word (a ``RuntimeError`` from
    ``raise_device_errors``, or from the next rasterizer call, which reads it too).
    Differentiable in ``table`` and in a tensor ``scale``.
    """
    _validate(table, codes, scale)
    gain = scale if isinstance(scale, torch.Tensor) else None
    scale = 1.0 if gain is not None else float(scale)
    if not torch.is_grad_enabled():
        return lookup_forward(table.contiguous(), codes.contiguous(), scale,
                              None if gain is None else gain.contiguous())
    return _CodebookLookup.apply(table, codes, scale, gain)
