"""Row operators around the fused linears: dropout, residual + dropout + RMS norm, rows in e4m3, and the GEMM that reads them.

They have no counterpart in the reference.  Eager calls go through compiled operators that bring their own autograd node
and argument checks (:func:`call_native`): their kernels take microseconds, and an ``autograd.Function`` in Python costs
more than that.  While ``torch.compile`` traces, or with ``CODA_B200_DISPATCH`` other than ``native``, the functions of
:mod:`coda_kernels_b200.functional` use the Python nodes over the custom ops below, with the same checks.
"""

from __future__ import annotations

import re
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from ._lib import CodaB200Error, check, lib
from .ops import _aligned16, _native, _noop_fake, _require, _stream, status_word

_DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
E4M3 = torch.float8_e4m3fn


_native_ops: dict = {}
_REFUSED = re.compile(r" failed \(code -?\d+\): ")  # how the dispatch layer reports a library call's status, as ``check`` does


def call_native(name: str, *args):
    """An operator of the compiled dispatch layer; what the library refuses is raised as the package's own exception, all else
    (a refused argument, no memory, a CUDA error) as it is."""
    op = _native_ops.get(name)
    if op is None:
        op = _native_ops[name] = getattr(torch.ops.coda_b200n, name).default
    try:
        return op(*args)
    except RuntimeError as ex:
        text = str(ex).split("\n")[0]
        if type(ex) is RuntimeError and _REFUSED.search(text):
            raise CodaB200Error(text) from ex
        raise


def apart(*tensors: Tensor) -> tuple[Tensor, ...]:
    """The tensors, one that is given again as a view of itself.  A traced ``autograd.Function`` that receives one tensor twice gets
    the gradient of its first place only."""
    return tuple(t.view_as(t) if any(t is u for u in tensors[:i]) else t for i, t in enumerate(tensors))


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _low_like(x: Tensor) -> Tensor:
    """Room for the bits of ``h`` below its type, four an element: ``coda_b200_add_rmsnorm_low_bytes``."""
    cols = x.shape[-1]
    rows = x.numel() // cols
    return x.new_empty(rows * cols // 8 if cols % 8 == 0 else (rows * cols + 7) // 8 + rows, dtype=torch.int32)


def _dense16(t: Optional[Tensor]) -> Optional[Tensor]:
    """What the row kernels take: dense and 16-byte aligned (a view that starts elsewhere is copied)."""
    return None if t is None else _aligned16(t)


# ------------------------------------------------------------------------------------------------ custom ops
@torch.library.custom_op("coda_b200::dropout_out", mutates_args=("out", "used"), device_types="cuda")
def _dropout_out(x: Tensor, p: float, rng: Optional[Tensor], stream_id: int, out: Tensor, used: Tensor) -> None:
    x = _dense16(x)
    cols = x.shape[-1]
    check(
        lib.coda_b200_dropout(x.data_ptr(), out.data_ptr(), x.numel() // cols, cols, _DTYPE_CODES[x.dtype], float(p), _ptr(rng), stream_id,
                              used.data_ptr(), _stream(x)),
        "dropout",
    )


@torch.library.custom_op("coda_b200::add_rmsnorm_out", mutates_args=("h", "low", "out", "rstd", "used"), device_types="cuda")
def _add_rmsnorm_out(x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float, p: float, rng: Optional[Tensor], stream_id: int,
                     h: Optional[Tensor], low: Optional[Tensor], out: Tensor, rstd: Tensor, used: Optional[Tensor]) -> None:
    x, residual, weight = _dense16(x), _dense16(residual), _dense16(weight)
    cols = x.shape[-1]
    check(
        lib.coda_b200_add_rmsnorm_fwd_low(x.data_ptr(), _ptr(residual), weight.data_ptr(), float(eps), float(p), _ptr(rng), stream_id,
                                          _ptr(used), _ptr(h), _ptr(low), out.data_ptr(), rstd.data_ptr(), x.numel() // cols, cols,
                                          _DTYPE_CODES[x.dtype], _stream(x)),
        "add_rmsnorm",
    )


@torch.library.custom_op("coda_b200::add_rmsnorm_bwd_out", mutates_args=("dx", "dres", "dweight"), device_types="cuda")
def _add_rmsnorm_bwd_out(dout: Tensor, dh: Optional[Tensor], h: Tensor, low: Optional[Tensor], rstd: Tensor, weight: Tensor, p: float,
                         rng: Optional[Tensor], stream_id: int, dx: Optional[Tensor], dres: Optional[Tensor],
                         dweight: Optional[Tensor]) -> None:
    dout, dh, h, low, weight = _dense16(dout), _dense16(dh), _dense16(h), _dense16(low), _dense16(weight)
    cols = h.shape[-1]
    rows = h.numel() // cols
    scratch_bytes = int(lib.coda_b200_add_rmsnorm_bwd_scratch_bytes(rows, cols)) if dweight is not None else 0
    scratch = torch.empty(scratch_bytes // 4, dtype=torch.float32, device=h.device) if dweight is not None else None
    check(
        lib.coda_b200_add_rmsnorm_bwd_low(dout.data_ptr(), _ptr(dh), h.data_ptr(), _ptr(low), rstd.data_ptr(), weight.data_ptr(), float(p),
                                          _ptr(rng), stream_id, _ptr(dx), _ptr(dres), _ptr(dweight), _ptr(scratch), scratch_bytes, rows,
                                          cols, _DTYPE_CODES[h.dtype], _stream(h)),
        "add_rmsnorm backward",
    )


@torch.library.custom_op("coda_b200::rows_e4m3_out", mutates_args=("h", "q", "scale"), device_types="cuda")
def _rows_e4m3_out(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float, h: Optional[Tensor], q: Tensor,
                   scale: Tensor) -> None:
    x, residual, weight = _dense16(x), _dense16(residual), _dense16(weight)
    cols = x.shape[-1]
    check(
        lib.coda_b200_rows_e4m3(x.data_ptr(), _ptr(residual), _ptr(weight), float(eps), _ptr(h), q.data_ptr(), scale.data_ptr(),
                                x.numel() // cols, cols, _DTYPE_CODES[x.dtype], _stream(x)),
        "rows_e4m3",
    )


@torch.library.custom_op("coda_b200::gemm_e4m3_out", mutates_args=("out",), device_types="cuda")
def _gemm_e4m3_out(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, out: Tensor) -> None:
    x, weight = _dense16(x), _dense16(weight)
    M, K = x.shape
    N = weight.shape[0]
    ws_bytes = int(lib.coda_b200_gemm_e4m3_workspace_bytes(M, N, K))
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=x.device) if ws_bytes > 0 else None
    check(
        lib.coda_b200_gemm_e4m3(x.data_ptr(), x_scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(), out.data_ptr(), N,
                                int(out.dtype == torch.float32), M, N, K, _ptr(ws), ws_bytes, status_word(x.device).data_ptr(), _stream(x)),
        "gemm_e4m3",
    )


for _op in (_dropout_out, _add_rmsnorm_out, _add_rmsnorm_bwd_out, _rows_e4m3_out, _gemm_e4m3_out):
    _op.register_fake(_noop_fake)


# ------------------------------------------------------------------------------------------------ compiled operators on fake tensors
def _like(x: Tensor) -> Tensor:
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _rows_like(x: Tensor) -> Tensor:
    return x.new_empty(x.numel() // x.shape[-1], dtype=torch.float32)


if _native is not None:

    @torch.library.register_fake("coda_b200n::dropout")
    def _(x, p, rng, stream):
        return _like(x)

    @torch.library.register_fake("coda_b200n::dropout_fwd")
    def _(x, p, rng, stream):
        return _like(x), x.new_empty(2, dtype=torch.int64)

    @torch.library.register_fake("coda_b200n::norm_fwd")
    def _(x, residual, weight, eps, p, rng, stream, keep_low):
        h = None if residual is None else _like(x)
        low = _low_like(x) if keep_low and h is not None and x.dtype.itemsize == 2 else None
        return _like(x), h, _rows_like(x), x.new_empty(2, dtype=torch.int64) if p > 0.0 else None, low

    @torch.library.register_fake("coda_b200n::norm_bwd")
    def _(dout, dh, h, low, rstd, weight, p, rng, stream, need_dx, need_dres, need_dw):
        return _like(h) if need_dx else None, _like(h) if need_dres else None, _like(weight) if need_dw else None

    @torch.library.register_fake("coda_b200n::rms_norm")
    def _(x, weight, eps):
        return _like(x)

    @torch.library.register_fake("coda_b200n::add_rms_norm")
    def _(x, residual, weight, eps, p, rng, stream):
        return _like(x), _like(x)

    @torch.library.register_fake("coda_b200n::rows_e4m3")
    def _(x, residual, weight, eps):
        scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
        return x.new_empty(x.shape, dtype=E4M3), scale, None if residual is None else _like(x)

    @torch.library.register_fake("coda_b200n::linear_e4m3")
    def _(x, x_scale, weight, weight_scale, out_fp32, status):
        return x.new_empty(x.shape[0], weight.shape[0], dtype=torch.float32 if out_fp32 else torch.bfloat16)


# ------------------------------------------------------------------------------------------------ argument checks
def _require_rows(x: Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError("coda_b200 operators run on CUDA tensors only; there is no CPU fallback")
    if x.dtype not in _DTYPE_CODES:
        raise NotImplementedError(f"coda_b200 row operators take bfloat16, float16 or float32, got {x.dtype}")
    _require(x.dim() >= 1 and x.shape[-1] > 0, "x must have a last dimension of at least one element")


def _require_like(t: Tensor, x: Tensor, name: str) -> None:
    _require(t.shape == x.shape and t.dtype == x.dtype and t.device == x.device, f"{name} must match x in shape, dtype and device")


def _require_weight(weight: Tensor, x: Tensor) -> None:
    _require(weight.dim() == 1 and weight.shape[0] == x.shape[-1] and weight.dtype == x.dtype and weight.device == x.device,
             "weight must hold one entry per column of x, in x's dtype, on x's device")


def _require_dropout(x: Tensor, p: float, rng: Optional[Tensor], stream: int) -> None:
    _require(0.0 <= p < 1.0, f"the dropout probability must be at least 0 and below 1, got {p}")
    _require(0 <= stream < 2**32, "the dropout stream must be a 32-bit number")
    _require(p == 0.0 or rng is not None, "dropout needs rng, an int64 CUDA tensor [seed, step]")
    if rng is not None:
        _require(rng.dtype == torch.int64 and rng.device == x.device and tuple(rng.shape) == (2,),
                 "rng must be an int64 tensor [seed, step] on x's device")


def _require_first_order(name: str) -> None:
    """Called by the backwards: autograd runs them with gradients enabled only to differentiate them in turn."""
    if not torch.compiler.is_compiling() and torch.is_grad_enabled():
        raise RuntimeError(f"{name} can be differentiated once only")


def _require_no_grad(name: str, *tensors: Optional[Tensor]) -> None:
    if not torch.compiler.is_compiling() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no backward: call it under torch.no_grad() or on detached tensors")


# ------------------------------------------------------------------------------------------------ wrappers (dense tensors)
def dropout_rows(x: Tensor, p: float, rng: Optional[Tensor], stream: int) -> tuple[Tensor, Tensor]:
    """``(out, used)``: dropout of a dense tensor and the ``[seed, step]`` its mask was made from."""
    out = torch.empty_like(x)
    used = torch.empty(2, dtype=torch.int64, device=x.device)
    _dropout_out(x, p, rng, stream, out, used)
    return out, used


def add_rmsnorm_forward(x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float, p: float, rng: Optional[Tensor], stream: int):
    """``(out, h or None, rstd, used or None, low or None)``; ``h`` is ``None`` when it would be ``x`` itself, ``low`` holds the bits
    of ``h`` below a 2-byte type."""
    out = torch.empty_like(x)
    h = torch.empty_like(x) if residual is not None or p > 0.0 else None
    rstd = torch.empty(x.numel() // x.shape[-1], dtype=torch.float32, device=x.device)
    used = torch.empty(2, dtype=torch.int64, device=x.device) if p > 0.0 else None
    low = _low_like(x) if h is not None and x.dtype.itemsize == 2 else None
    _add_rmsnorm_out(x, residual, weight, eps, p, rng, stream, h, low, out, rstd, used)
    return out, h, rstd, used, low


def add_rmsnorm_backward(dout: Tensor, dh: Optional[Tensor], h: Tensor, low: Optional[Tensor], rstd: Tensor, weight: Tensor, p: float,
                         rng: Optional[Tensor], stream: int, need_dx: bool, need_dres: bool, need_dw: bool):
    """``(dx, dresidual, dweight)``, ``None`` where not wanted."""
    dx = torch.empty_like(h) if need_dx else None
    dres = torch.empty_like(h) if need_dres else None
    dw = None
    if need_dw:
        dw = torch.empty_like(weight) if h.numel() > 0 else torch.zeros_like(weight)
    _add_rmsnorm_bwd_out(dout, dh, h, low, rstd, weight, p, rng, stream, dx, dres, dw)
    return dx, dres, dw


def rows_e4m3(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float):
    """``(q, scale, h or None)``: rows of ``x`` (plus ``residual``, normalised with ``weight``) as e4m3 values and scales."""
    h = torch.empty_like(x) if residual is not None else None
    q = torch.empty(x.shape, dtype=E4M3, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _rows_e4m3_out(x, residual, weight, eps, h, q, scale)
    return q, scale, h


def gemm_e4m3(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``(x * x_scale[:, None]) @ (weight * weight_scale[:, None])^T`` for dense e4m3 ``x [M, K]`` and ``weight [N, K]``."""
    for t in (x, x_scale, weight, weight_scale):
        if not t.is_cuda:
            raise RuntimeError("coda_b200 operators run on CUDA tensors only; there is no CPU fallback")
        _require(t.device == x.device, "all operands must be on one device")
    if x.dtype != E4M3 or weight.dtype != E4M3:
        raise NotImplementedError(f"x and weight must be float8_e4m3fn, got {x.dtype} and {weight.dtype}")
    _require(x.dim() == 2 and weight.dim() == 2 and x.shape[1] == weight.shape[1], "x [M, K] and weight [N, K] expected")
    _require(x.shape[1] > 0 and x.shape[1] % 16 == 0, "K must be a positive multiple of 16")
    _require(weight.shape[0] > 0 and weight.shape[0] % 8 == 0, "the number of weight rows must be a positive multiple of 8")
    for name, s, n in (("x_scale", x_scale, x.shape[0]), ("weight_scale", weight_scale, weight.shape[0])):
        _require(s.dtype == torch.float32 and tuple(s.shape) == (n,), f"{name} must be float32 with one entry per row")
    x, x_scale, weight, weight_scale = x.contiguous(), x_scale.contiguous(), weight.contiguous(), weight_scale.contiguous()
    out = torch.empty(x.shape[0], weight.shape[0], dtype=out_dtype, device=x.device)
    if x.shape[0] > 0:
        _gemm_e4m3_out(x, x_scale, weight, weight_scale, out)
    return out
