"""``linear_cross_entropy_pieces``: the LM-head loss for batches whose ``[M, V]`` gradient buffer would not fit.

An extension with no counterpart in the reference.  :func:`linear_cross_entropy` keeps ``softmax - onehot`` of the whole
batch, ``2 M V`` bytes, from forward to backward.  Here the node keeps the rows' log-sum-exp, and with the rows that count put
first their labels and positions (4 bytes a row each), beside the caller's tensors; the backward walks the vocabulary in pieces, computes each piece's logits again and turns them into its part of the two
gradients.  The price is that one product (a third more work in the backward); what it saves is everything of size
``M V`` but one ``[M, piece]`` buffer during the backward.

Ignored rows may hold anything.  They have no part in the products where those are large enough to be worth it: the rows that
count are first put together on the device, and the products end where they end, without the host knowing where that is.
"""

from __future__ import annotations

from typing import Optional

import torch

from .._guards import autocast_custom_bwd, autocast_custom_fwd, input_guard
from ..ops import _debug_check_targets, _fast, _require, lazy_status_check, status_word
from ..ops_ce import ce_pieces_backward, ce_pieces_forward, default_piece
from ..ops_rows import _require_first_order, apart, call_native


class LinearCrossEntropyPieces(torch.autograd.Function):
    """Saves ``x``, the weight, the labels (those of the rows that count first, with the positions), the log-sum-exp and
    ``inv_count``."""

    @staticmethod
    @input_guard
    @autocast_custom_fwd
    def forward(ctx, x, weight, target, ignore_index: int, reduction: str, piece: int) -> torch.Tensor:
        loss, inv_count, lse, labels, position, live = ce_pieces_forward(x, weight, target, ignore_index, reduction == "mean")
        ctx.save_for_backward(x, weight, labels, lse, inv_count, position, live)
        ctx.ignore_index, ctx.piece = ignore_index, piece
        return loss

    @staticmethod
    @input_guard
    @autocast_custom_bwd
    def backward(ctx, dloss: torch.Tensor):
        _require_first_order("linear_cross_entropy_pieces")
        x, weight, labels, lse, inv_count, position, live = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[:2]
        return (*ce_pieces_backward(dloss, inv_count, lse, x, weight, labels, position, live, ctx.ignore_index, ctx.piece, need_dx,
                                    need_dw), None, None, None, None)


def linear_cross_entropy_pieces(
    x: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor,
    ignore_index: int = -100,
    reduction: str = "mean",
    piece: Optional[int] = None,
) -> torch.Tensor:
    """``x [M, K]``, ``weight [V, K]`` (any ``V``), int32 ``target [M]`` -> the scalar loss of ``linear_cross_entropy``.

    ``piece`` is the number of vocabulary columns the backward works on at once (default: as many as make its buffer
    512 MiB, at least 8192).  A label outside ``[0, V)`` that is not ``ignore_index`` makes the loss, its row of
    ``dx`` and ``dweight`` NaN; ``"mean"`` over no label at all is NaN, with gradients of zero."""
    assert reduction in ("mean", "sum")
    assert target.dtype == torch.int32
    _require(x.dim() == 2 and weight.dim() == 2, "x [M, K] and weight [V, K] expected")
    if piece is None:
        piece = default_piece(x.shape[0], weight.shape[0])
    _require(piece >= 1, "piece must be at least 1")
    if _fast() and x.is_cuda:
        lazy_status_check(x.device)
        _debug_check_targets(target, weight.shape[0], ignore_index)
        return call_native("linear_cross_entropy_pieces", x, weight, target, ignore_index, reduction == "mean", int(piece), status_word(x.device))
    return LinearCrossEntropyPieces.apply(*apart(x, weight), target, ignore_index, reduction, int(piece))
