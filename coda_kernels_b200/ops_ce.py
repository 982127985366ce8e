"""Cross entropy over a vocabulary walked in pieces, keeping no logits between forward and backward.

It has no counterpart in the reference.  Eager calls run the compiled form of the same sequence (see
:mod:`coda_kernels_b200.ops_rows`); what is here serves ``torch.compile`` and the other dispatch modes.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import ops
from ._lib import check, lib
from .ops import _aligned16, _native, _noop_fake, _require, _require_cuda_bf16, _stream, lse_tiles, status_word


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


# The ops below copy a matrix of the caller's that does not start on a 16-byte boundary, as the compiled form does: only here, where
# they run, are addresses known (a tracer has none).


@torch.library.custom_op("coda_b200::ce_loss_out", mutates_args=("parts", "lse", "loss", "inv_count"), device_types="cuda")
def _ce_loss_out(x: Tensor, weight: Tensor, target: Tensor, ignore_index: int, mean: bool, live: Optional[Tensor], parts: Tensor,
                 lse: Tensor, loss: Tensor, inv_count: Tensor) -> None:
    x, weight = _aligned16(x), _aligned16(weight)
    M, K = x.shape
    V = weight.shape[0]
    tiles = lse_tiles(V)
    base = parts.data_ptr()
    check(
        lib.coda_b200_ce_loss(x.data_ptr(), K, 1, weight.data_ptr(), 1, K, target.data_ptr(), ignore_index, int(mean), _ptr(live), base,
                              base + 4 * M * tiles, base + 8 * M * tiles, lse.data_ptr(), base + 8 * M * tiles + 4 * M, loss.data_ptr(), inv_count.data_ptr(), M, V,
                              K, status_word(x.device).data_ptr(), _stream(x)),
        "ce_loss",
    )


@torch.library.custom_op("coda_b200::gemm_softmax_grad_out", mutates_args=("grad",), device_types="cuda")
def _gemm_softmax_grad_out(x: Tensor, weight: Tensor, lse: Tensor, target: Tensor, ignore_index: int, col0: int, live: Optional[Tensor],
                           grad: Tensor) -> None:
    x, weight = _aligned16(x), _aligned16(weight)
    M, K = x.shape
    N = weight.shape[0]
    check(
        lib.coda_b200_gemm_softmax_grad(x.data_ptr(), K, 1, weight.data_ptr(), 1, K, lse.data_ptr(), target.data_ptr(), ignore_index, col0,
                                        _ptr(live), grad.data_ptr(), grad.shape[1], M, N, K, status_word(x.device).data_ptr(), _stream(x)),
        "gemm_softmax_grad",
    )


@torch.library.custom_op("coda_b200::ce_compact_out", mutates_args=("position", "labels", "live", "rows"), device_types="cuda")
def _ce_compact_out(x: Tensor, target: Tensor, ignore_index: int, position: Tensor, labels: Tensor, live: Tensor, rows: Tensor) -> None:
    x = _aligned16(x)
    check(
        lib.coda_b200_ce_compact(x.data_ptr(), target.data_ptr(), ignore_index, position.data_ptr(), labels.data_ptr(), live.data_ptr(),
                                 rows.data_ptr(), x.shape[0], x.shape[1], _stream(x)),
        "ce_compact",
    )


@torch.library.custom_op("coda_b200::ce_gather_out", mutates_args=("rows",), device_types="cuda")
def _ce_gather_out(x: Tensor, position: Tensor, live: Tensor, rows: Tensor) -> None:
    x = _aligned16(x)
    check(lib.coda_b200_ce_gather(x.data_ptr(), position.data_ptr(), live.data_ptr(), rows.data_ptr(), x.shape[0], x.shape[1], _stream(x)),
          "ce_gather")


@torch.library.custom_op("coda_b200::ce_mask_out", mutates_args=("rows",), device_types="cuda")
def _ce_mask_out(x: Tensor, target: Tensor, ignore_index: int, rows: Tensor) -> None:
    x = _aligned16(x)
    check(lib.coda_b200_ce_mask(x.data_ptr(), target.data_ptr(), ignore_index, rows.data_ptr(), x.shape[0], x.shape[1], _stream(x)), "ce_mask")


@torch.library.custom_op("coda_b200::ce_scatter_out", mutates_args=("dx",), device_types="cuda")
def _ce_scatter_out(rows: Tensor, position: Tensor, dx: Tensor) -> None:
    check(lib.coda_b200_ce_scatter(rows.data_ptr(), position.data_ptr(), dx.data_ptr(), rows.shape[0], rows.shape[1], _stream(rows)), "ce_scatter")


@torch.library.custom_op("coda_b200::gemm_ragged_out", mutates_args=("out",), device_types="cuda")
def _gemm_ragged_out(A: Tensor, B: Tensor, C: Optional[Tensor], alpha: Tensor, out: Tensor) -> None:
    """``out = alpha A @ B (+ C)`` for operands of any contiguous extent; ``C`` is fp32 and laid out as ``out``."""
    _gemm_ragged(A, B, C, alpha, out)


def _gemm_ragged(A: Tensor, B: Tensor, C: Optional[Tensor], alpha: Tensor, out: Tensor) -> None:
    B = _aligned16(B)
    (M, K), N = A.shape, B.shape[1]
    ws_bytes = int(lib.coda_b200_gemm_workspace_bytes(M, N, K)) if C is None else 0
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=A.device) if ws_bytes > 0 else None
    check(
        lib.coda_b200_gemm_ragged(A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0), B.stride(1), _ptr(C), out.data_ptr(),
                                  out.stride(0), int(out.dtype == torch.float32), M, N, K, alpha.data_ptr(), _ptr(ws), ws_bytes,
                                  status_word(A.device).data_ptr(), _stream(A)),
        "gemm_ragged",
    )


@torch.library.custom_op("coda_b200::gemm_live_out", mutates_args=("out",), device_types="cuda")
def _gemm_live_out(grad: Tensor, n: int, B: Tensor, C: Optional[Tensor], alpha: Tensor, live: Tensor, along_depth: bool, out: Tensor) -> None:
    """``grad[:, :n] @ B`` over the counted rows, or ``grad[:, :n]^T @ B`` summed over them."""
    B = _aligned16(B)
    M, N = grad.shape[0], B.shape[1]
    if not along_depth and C is None and lib.coda_b200_gemm_workspace_bytes(M, N, n) > 0:  # few tiles, cut along the contraction: all rows
        _gemm_ragged(grad[:, :n], B, None, alpha, out)
        return
    check(
        lib.coda_b200_gemm_live(grad.data_ptr(), grad.shape[1], B.data_ptr(), N, _ptr(C), out.data_ptr(), N, int(out.dtype == torch.float32),
                                alpha.data_ptr(), live.data_ptr(), int(along_depth), n if along_depth else M, N, M if along_depth else n,
                                status_word(B.device).data_ptr(), _stream(B)),
        "gemm_live",
    )


@torch.library.custom_op("coda_b200::ce_alpha_out", mutates_args=("alpha",), device_types="cuda")
def _ce_alpha_out(dloss: Tensor, inv_count: Tensor, alpha: Tensor) -> None:
    check(lib.coda_b200_ce_alpha(dloss.data_ptr(), inv_count.data_ptr(), alpha.data_ptr(), _stream(alpha)), "ce_alpha")


for _op in (_ce_loss_out, _ce_alpha_out, _gemm_softmax_grad_out, _ce_compact_out, _ce_gather_out, _ce_mask_out, _ce_scatter_out, _gemm_ragged_out, _gemm_live_out):
    _op.register_fake(_noop_fake)


if _native is not None:  # the compiled operators on fake tensors

    @torch.library.register_fake("coda_b200n::linear_cross_entropy_pieces")
    def _(x, weight, target, ignore_index, mean, piece, status):
        return x.new_empty((), dtype=torch.float32)

    @torch.library.register_fake("coda_b200n::ce_pieces_fwd")
    def _(x, weight, target, ignore_index, mean, compact, status):
        f32 = dict(dtype=torch.float32)
        rows = [target.new_empty(n) for n in (x.shape[0], x.shape[0], 1)] if compact else [None] * 3
        return x.new_empty((), **f32), x.new_empty((), **f32), x.new_empty(x.shape[0], **f32), *rows

    @torch.library.register_fake("coda_b200n::ce_pieces_bwd")
    def _(dloss, inv_count, lse, x, weight, target, position, live, ignore_index, piece, need_dx, need_dw, status):
        return x.new_empty(x.shape) if need_dx else None, weight.new_empty(weight.shape) if need_dw else None


# Default size of the [rows, piece] gradient buffer, in elements (512 MiB), and the narrowest piece it is cut down to for
# very many rows: below it the fp32 sum of dx, read and written once a piece, would cost more than a few percent of the
# piece's GEMMs.
_PIECE_ELEMENTS = 1 << 28
_PIECE_MIN = 8192


def default_piece(rows: int, vocab: int) -> int:
    """Columns per piece: pieces of one width, a multiple of the GEMM's column tile, as few as the buffer allows."""
    widest = max(_PIECE_MIN, _PIECE_ELEMENTS // max(rows, 1))
    pieces = -(-vocab // widest)
    return min(vocab, -(-vocab // pieces // 256) * 256) if pieces > 1 else vocab


def _require_ce(x: Tensor, weight: Tensor, target: Tensor, ignore_index: int) -> None:
    _require_cuda_bf16(x, weight)
    _require(x.dim() == 2 and weight.dim() == 2 and x.shape[1] == weight.shape[1], "x [M, K] and weight [V, K] expected")
    _require(weight.shape[0] > 0 and x.shape[1] > 0 and x.shape[1] % 8 == 0, "weight must have rows, and K must be a positive multiple of 8")
    _require(target.device == x.device and weight.device == x.device, "x, weight and target must be on one device")
    _require(tuple(target.shape) == (x.shape[0],), "target must have one label per row")
    _require(-(2**31) <= ignore_index < 2**31, "ignore_index must fit int32")


@torch.compiler.assume_constant_result
def _options_allow_compacting() -> bool:
    return bool(lib.coda_b200_ce_compacts(1 << 20, 1 << 20, 1 << 10))


def _compacts(M: int, V: int, K: int) -> bool:
    """``coda_b200_ce_compacts`` in a form that can be traced.  A compiled program keeps the options it was traced with."""
    return M > 0 and V >= 8192 and 2 * M * V * K >= 50_000_000_000 and _options_allow_compacting()


def ce_pieces_forward(x: Tensor, weight: Tensor, target: Tensor, ignore_index: int, mean: bool):
    """``(loss, inv_count, lse, labels, position, live)``; nothing of size ``[M, V]`` is written.  ``labels`` and ``lse`` are in the
    order of the rows, or, where that pays, those of the rows that count come first (``live`` of them, from ``position``)."""
    _require_ce(x, weight, target, ignore_index)
    ops._debug_check_targets(target, weight.shape[0], ignore_index)
    M = x.shape[0]
    f32 = dict(dtype=torch.float32, device=x.device)
    if M == 0:  # a sum over nothing, and 0 / 0
        return (torch.full((), float("nan") if mean else 0.0, **f32), torch.zeros((), **f32),
                torch.empty(0, **f32), target, None, None)
    position = live = None
    if _compacts(M, weight.shape[0], x.shape[1]):
        rows, labels, position = torch.empty_like(x), torch.empty_like(target), torch.empty_like(target)
        live = torch.empty(1, dtype=torch.int32, device=x.device)
        _ce_compact_out(x, target, ignore_index, position, labels, live, rows)
        x, target = rows, labels
    parts = torch.empty(2 * M * lse_tiles(weight.shape[0]) + 2 * M, **f32)
    lse, loss, inv_count = torch.empty(M, **f32), torch.empty((), **f32), torch.empty((), **f32)
    _ce_loss_out(x, weight, target, ignore_index, mean, live, parts, lse, loss, inv_count)
    return loss, inv_count, lse, target, position, live


def ce_pieces_backward(dloss: Tensor, inv_count: Tensor, lse: Tensor, x: Tensor, weight: Tensor, target: Tensor, position: Optional[Tensor],
                       live: Optional[Tensor], ignore_index: int, piece: int, need_dx: bool,
                       need_dw: bool) -> tuple[Optional[Tensor], Optional[Tensor]]:
    """Gradients from one ``[M, piece]`` buffer: per piece of the vocabulary its softmax gradient ``g`` (the logits are
    computed again), its rows of ``dweight = alpha g^T x``, and ``dx += alpha g @ weight`` in fp32."""
    M, K = x.shape
    V = weight.shape[0]
    if M == 0:
        return (torch.zeros_like(x) if need_dx else None), (torch.zeros_like(weight) if need_dw else None)
    alpha = torch.empty(1, dtype=torch.float32, device=x.device)
    _ce_alpha_out(dloss.to(torch.float32), inv_count, alpha)
    width = min(piece, V)
    if live is not None:  # (the node does not keep this copy: it is small beside the products, but not beside what the node keeps)
        rows = torch.empty_like(x)
        _ce_gather_out(x, position, live, rows)
        x = rows
    g = torch.empty(M, -(-width // 8) * 8, dtype=x.dtype, device=x.device)
    dx = torch.empty_like(x) if need_dx else None
    dw = torch.empty_like(weight) if need_dw else None
    dx32 = torch.empty(M, K, dtype=torch.float32, device=x.device) if need_dx and width < V else None
    counted = x  # the rows of the weight gradient: whatever an ignored row holds has no part in it
    if need_dw and live is None:
        counted = torch.empty_like(x)
        _ce_mask_out(x, target, ignore_index, counted)
    for c0 in range(0, V, width):
        n = min(width, V - c0)
        w = weight[c0:c0 + n]
        _gemm_softmax_grad_out(x, w, lse, target, ignore_index, c0, live, g)
        sum_so_far = dx32 if c0 > 0 else None
        if live is None:
            gp = g[:, :n]
            if need_dw:
                _gemm_ragged_out(gp.mT, counted, None, alpha, dw[c0:c0 + n])
            if need_dx:
                _gemm_ragged_out(gp, w, sum_so_far, alpha, dx32 if c0 + n < V else dx)
        else:
            if need_dw:
                _gemm_live_out(g, n, x, None, alpha, live, True, dw[c0:c0 + n])
            if need_dx:
                _gemm_live_out(g, n, w, sum_so_far, alpha, live, False, dx32 if c0 + n < V else dx)
    if need_dx and live is not None:  # into the memory of the rows, which are not needed any more
        _ce_scatter_out(dx, position, x)
        dx = x
    return dx, dw
