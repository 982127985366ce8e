"""``rms_norm`` / ``add_rms_norm``: what stands between two fused linears, in one pass each way; and its 8-bit outputs.

Extensions with no counterpart in the reference, whose norms live inside the fused layer blocks.
``add_rms_norm`` ends a sublayer: ``h = residual + dropout(x)`` is the new residual stream and ``out`` its RMS norm, the
next linear's input.  The statistic and ``out`` come from the unrounded ``h``; the backward works from the stored one, from the
bits of ``h`` below a 2-byte type (half a byte an element, without which ``dweight`` carries the rounding of ``h`` beside its own)
and from ``rstd``, and makes the dropout mask again.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from .._guards import autocast_custom_bwd, autocast_custom_fwd, input_guard
from ..ops import _fast, _require
from ..ops_rows import (
    _require_dropout,
    _require_first_order,
    _require_like,
    _require_no_grad,
    _require_rows,
    _require_weight,
    add_rmsnorm_backward,
    add_rmsnorm_forward,
    apart,
    call_native,
    rows_e4m3,
)


class RMSNorm(torch.autograd.Function):
    """Saves ``(x, weight, rstd)``."""

    @staticmethod
    @input_guard
    @autocast_custom_fwd
    def forward(ctx, x: Tensor, weight: Tensor, eps: float) -> Tensor:
        _require_rows(x)
        _require_weight(weight, x)
        out, _, rstd, _, _ = add_rmsnorm_forward(x, None, weight, eps, 0.0, None, 0)
        ctx.save_for_backward(x, weight, rstd)
        return out

    @staticmethod
    @input_guard
    @autocast_custom_bwd
    def backward(ctx, dout: Tensor):
        _require_first_order("rms_norm")
        x, weight, rstd = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[:2]
        _, dx, dw = add_rmsnorm_backward(dout, None, x, None, rstd, weight, 0.0, None, 0, False, need_dx, need_dw)
        return dx, dw, None


class AddRMSNorm(torch.autograd.Function):
    """Saves ``(h, weight, rstd)``, the bits below ``h`` and the 16 bytes the dropout mask was made from."""

    @staticmethod
    @input_guard
    @autocast_custom_fwd
    def forward(ctx, x: Tensor, residual: Tensor, weight: Tensor, eps: float, p: float, rng: Optional[Tensor], stream: int):
        _require_rows(x)
        _require_like(residual, x, "residual")
        _require_weight(weight, x)
        _require_dropout(x, p, rng, stream)
        out, h, rstd, used, low = add_rmsnorm_forward(x, residual, weight, eps, p, rng, stream)
        ctx.save_for_backward(h, weight, rstd, used, low)
        ctx.p, ctx.stream = p, stream
        ctx.set_materialize_grads(False)
        return out, h

    @staticmethod
    @input_guard
    @autocast_custom_bwd
    def backward(ctx, dout: Optional[Tensor], dh: Optional[Tensor]):
        _require_first_order("add_rms_norm")
        h, weight, rstd, used, low = ctx.saved_tensors
        need_dx, need_dres, need_dw = ctx.needs_input_grad[:3]
        if dout is None:  # only h was used
            dout = torch.zeros_like(h)
        dx, dres, dw = add_rmsnorm_backward(dout, dh, h, low, rstd, weight, ctx.p, used, ctx.stream, need_dx, need_dres, need_dw)
        return dx, dres, dw, None, None, None, None


def rms_norm(x: Tensor, weight: Tensor, eps: float) -> Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last dimension of ``x [..., N]`` (bf16, fp16 or fp32)."""
    if _fast() and x.is_cuda:
        return call_native("rms_norm", x, weight, eps)
    return RMSNorm.apply(*apart(x, weight), float(eps))


def add_rms_norm(x: Tensor, residual: Tensor, weight: Tensor, eps: float, p: float = 0.0, rng: Optional[Tensor] = None,
                 stream: int = 0) -> tuple[Tensor, Tensor]:
    """``(out, h)``: ``h = residual + dropout(x)`` and ``out = rms_norm(h, weight, eps)``, ``x`` and ``residual [..., N]``.

    ``p``, ``rng`` and ``stream`` are those of :func:`dropout`, and give the same mask."""
    if _fast() and x.is_cuda:
        return call_native("add_rms_norm", x, residual, weight, eps, p, rng, stream)
    return AddRMSNorm.apply(*apart(x, residual, weight), float(eps), float(p), rng, int(stream))


def _rows_e4m3(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float):
    if _fast() and x.is_cuda:
        return call_native("rows_e4m3", x, residual, weight, eps)
    _require_no_grad("the e4m3 output", x, residual, weight)
    return _rows_e4m3_composed(x, residual, weight, float(eps))


@input_guard
def _rows_e4m3_composed(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float):
    _require_rows(x)
    if residual is not None:
        _require_like(residual, x, "residual")
    if weight is not None:
        _require_weight(weight, x)
    return rows_e4m3(x, residual, weight, eps)


def rms_norm_e4m3(x: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    """``(q, scale)``: the rows of ``rms_norm(x, weight, eps)`` as ``float8_e4m3fn`` values and one fp32 scale each
    (``q * scale[..., None]`` is the row), for :func:`linear_e4m3`.  Inference only."""
    _require(weight is not None, "rms_norm_e4m3 needs a weight (quantize_e4m3 takes rows as they are)")
    q, scale, _ = _rows_e4m3(x, None, weight, eps)
    return q, scale


def add_rms_norm_e4m3(x: Tensor, residual: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor, Tensor]:
    """``(q, scale, h)``: :func:`add_rms_norm` without dropout, its first output in 8 bits.  Inference only."""
    _require(residual is not None and weight is not None, "add_rms_norm_e4m3 needs a residual and a weight")
    return _rows_e4m3(x, residual, weight, eps)


def quantize_e4m3(x: Tensor) -> tuple[Tensor, Tensor]:
    """``(q, scale)``: the rows of ``x [..., N]`` as ``float8_e4m3fn`` values and ``scale = max|row| / 448`` each: a
    weight, once, or activations that no norm precedes."""
    q, scale, _ = _rows_e4m3(x, None, None, 0.0)
    return q, scale
