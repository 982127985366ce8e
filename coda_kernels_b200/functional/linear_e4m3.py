"""``linear_e4m3``: the projection of rows in 8 bits by a weight in 8 bits, for inference.

An extension with no counterpart in the reference.  Both operands come from :func:`quantize_e4m3` or from a norm that
ends in 8 bits; the scales of the row and of the weight row multiply the fp32 accumulator once, in the epilogue.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from .._guards import input_guard
from ..ops import _fast, _require, lazy_status_check, status_word
from ..ops_rows import _require_no_grad, call_native, gemm_e4m3


@input_guard
def _linear_e4m3(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, out_dtype: torch.dtype) -> Tensor:
    return gemm_e4m3(x, x_scale, weight, weight_scale, out_dtype)


def linear_e4m3(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``x [M, K]``, ``weight [N, K]`` (``float8_e4m3fn``; K a multiple of 16, N of 8), ``x_scale [M]``, ``weight_scale [N]``
    -> ``(x * x_scale) @ (weight * weight_scale)^T`` as bf16 (default) or fp32.  Inference only."""
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    _require(out_dtype in (torch.bfloat16, torch.float32), "out_dtype must be bfloat16 or float32")
    if _fast() and x.is_cuda:
        lazy_status_check(x.device)
        return call_native("linear_e4m3", x, x_scale, weight, weight_scale, out_dtype == torch.float32, status_word(x.device))
    _require_no_grad("linear_e4m3", x, x_scale, weight, weight_scale)
    return _linear_e4m3(x, x_scale, weight, weight_scale, out_dtype)
