"""``dropout``: counter-based dropout whose mask is computed, never stored.

An extension with no counterpart in the reference.  Whether element ``(r, c)`` stays follows from
``(seed, step, stream, r, c)`` alone (Philox4x32-10), so the backward makes the same mask again instead of reading one,
any launch geometry gives the same bits, and a replayed CUDA graph draws a new mask once its ``step`` was advanced.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from .._guards import autocast_custom_bwd, autocast_custom_fwd, input_guard
from ..ops import _fast
from ..ops_rows import _require_dropout, _require_first_order, _require_rows, call_native, dropout_rows


class Dropout(torch.autograd.Function):
    """Saves the 16 bytes ``[seed, step]`` the forward read, so ``rng`` may advance before the backward."""

    @staticmethod
    @input_guard
    @autocast_custom_fwd
    def forward(ctx, x: Tensor, p: float, rng: Optional[Tensor], stream: int) -> Tensor:
        _require_rows(x)
        _require_dropout(x, p, rng, stream)
        out, used = dropout_rows(x, p, rng, stream)
        ctx.save_for_backward(used)
        ctx.p, ctx.stream = p, stream
        return out

    @staticmethod
    @input_guard
    @autocast_custom_bwd
    def backward(ctx, dout: Tensor):
        _require_first_order("dropout")
        (used,) = ctx.saved_tensors
        return dropout_rows(dout, ctx.p, used, ctx.stream)[0], None, None, None


def dropout(x: Tensor, p: float, rng: Optional[Tensor] = None, stream: int = 0) -> Tensor:
    """Zeroes each element of ``x [..., N]`` with probability ``p`` and multiplies the others by ``1 / (1 - p)``.

    ``rng`` is an int64 CUDA tensor ``[seed, step]`` (not needed for ``p = 0``); advance ``step`` (``rng[1] += 1``) once a
    training step, and give every place of the model its own ``stream`` number.  The mask depends on the rows and the
    last dimension of ``x``, not on its other dimensions."""
    if _fast() and x.is_cuda:
        return call_native("dropout", x, p, rng, stream)
    return Dropout.apply(x, float(p), rng, int(stream))
