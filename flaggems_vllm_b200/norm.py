"""RMS norm of the residual stream: ``rms_norm`` (differentiable), ``fused_add_rms_norm`` (in place) and
``rms_norm_quant`` (8-bit output with scales).

They stand in front of the MoE layer: the norm feeds the router and ``fused_experts_impl``, the 8-bit form the
projections that ``per_token_group_quant_fp8`` feeds otherwise."""

from __future__ import annotations

import logging
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .quant import SUPPORTED_FP8_DTYPE

logger = logging.getLogger(__name__)

_FORMATS = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1, torch.int8: 2}
_MAX_COLS, _MAX_ROWS, _MAX_EPS = 1 << 24, 0x7FFFFFFF, 3e38


def _check(x, weight, eps, residual, what):
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what}: x must have a last dimension to normalise")
    _lib.dtype_code(x.dtype)  # ValueError("Unsupported dtype")
    if x.shape[-1] > _MAX_COLS:
        raise ValueError(f"{what}: rows of at most {_MAX_COLS} elements")
    if x.numel() // x.shape[-1] > _MAX_ROWS:
        raise ValueError(f"{what}: at most {_MAX_ROWS} rows")
    if weight.ndim != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"{what}: weight must be [{x.shape[-1]}], got {list(weight.shape)}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{what}: weight must be of the type of x or float32, got {weight.dtype}")
    if not 0.0 <= eps < _MAX_EPS:
        raise ValueError(f"{what}: eps must be finite in fp32 and not negative")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{what}: residual must have the shape and type of x")
    _lib.require_cuda(x, what)
    for t in (weight, residual):
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: operands on different devices")


def _refused(what):
    raise _lib.MoeKernelError(f"{what}: the operands were not taken")


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    residual: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``weight * h / sqrt(mean(h ** 2) + eps)`` over the last dimension, in fp32, rounded once; returns it, or with a
    residual (it, h).

    ``h`` is ``x``, or ``x + residual`` rounded to their type: the stream as the next layer finds it.  ``weight`` has the
    type of ``x`` or float32.  Differentiable once in all three, backwards; the weight's gradient is summed in fp32, in the
    same order in every run.  The mean square is an fp32 number: rows whose mean square is beyond it are normed to zero, and
    below 2^-130 (with ``eps`` of no more) it loses bits."""
    logger.debug("GEMS RMS NORM")
    out = _lib.host().rms_norm(x, weight, eps, residual) if x.is_cuda else None
    if out is None:
        eps = float(eps)
        _check(x, weight, eps, residual, "rms_norm")
        out = _lib.host().rms_norm(x.contiguous(), weight.contiguous(), eps,
                                   None if residual is None else residual.contiguous())
        if out is None:
            _refused("rms_norm")
    return out


def fused_add_rms_norm(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """In place: ``residual`` becomes the stream ``x + residual``, ``x`` its norm; returns (x, residual).

    Values are those of ``rms_norm(x, weight, eps, residual)``.  The rows of both may lie in wider buffers, whose other
    columns stay as they are, with any number of dimensions in front at one row distance; neither may share memory with the
    other or with the weight.  Not differentiable: refused where a gradient is wanted."""
    logger.debug("GEMS FUSED ADD RMS NORM")
    if not x.is_cuda or not _lib.host().fused_add_rms_norm(x, residual, weight, eps):
        what, eps = "fused_add_rms_norm", float(eps)
        if residual is None:
            raise ValueError(f"{what}: there must be a residual")
        _check(x, weight, eps, residual, what)
        if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or weight.requires_grad):
            raise RuntimeError(f"{what} works in place and has no gradient: use rms_norm, or torch.no_grad()")
        if not _lib.host().fused_add_rms_norm(x, residual, weight.contiguous(), eps):
            raise ValueError(f"{what}: x and residual must be rows of contiguous elements that share no memory with each other "
                             "or the weight")
    return x, residual


def rms_norm_quant(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    residual: Optional[torch.Tensor] = None,
    group_size: Optional[int] = None,
    dtype: Optional[torch.dtype] = None,
    column_major_scales: bool = False,
    scale_ue8m0: bool = False,
    quant_eps: float = 1e-10,
    return_norm: bool = False,
) -> Tuple[torch.Tensor, ...]:
    """``rms_norm`` with its output in 8 bits: returns (x_q, x_s), then the stream ``h`` where there is a residual, then
    the norm itself where ``return_norm`` asks for it.

    ``x_s`` holds one scale per ``group_size`` elements of a row (None: one per row), shape
    ``x.shape[:-1] + (cols / group_size,)``, column-major in memory when ``column_major_scales``;
    ``x_s = max(amax, quant_eps) / qmax``; a scale of zero (``quant_eps=0``) stands over zeros.  ``scale_ue8m0`` raises
    scales below 1e-10 to it and rounds up to a power of two, as ``per_token_group_quant_fp8`` does: the smallest is
    2^-33, whatever ``quant_eps``.  ``dtype`` is float8_e4m3fn (default), float8_e5m2 or int8.  The fp32 value of the norm
    is quantised, not its 16-bit rounding.  A NaN makes its group's scale NaN.  Not differentiable: refused where a
    gradient is wanted."""
    logger.debug("GEMS RMS NORM QUANT")
    what = "rms_norm_quant"
    dtype = SUPPORTED_FP8_DTYPE if dtype is None else dtype
    if dtype not in _FORMATS:
        raise NotImplementedError(f"{what}: 8-bit format {dtype} is not implemented (e4m3fn, e5m2 and int8 are)")
    group = 0 if group_size is None else group_size
    flags = int(bool(column_major_scales)) | (2 if scale_ue8m0 else 0)
    args = (group, _FORMATS[dtype], quant_eps, flags, bool(return_norm))
    out = _lib.host().rms_norm_quant(x, weight, eps, residual, *args) if x.is_cuda and group_size != 0 else None
    if out is None:
        eps, quant_eps = float(eps), float(quant_eps)
        _check_quant(x, group_size, dtype, column_major_scales, scale_ue8m0, quant_eps, what)
        _check(x, weight, eps, residual, what)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
            raise RuntimeError(f"{what} has no gradient: use rms_norm, or torch.no_grad()")
        out = _lib.host().rms_norm_quant(x.contiguous(), weight.contiguous(), eps,
                                         None if residual is None else residual.contiguous(), int(group), _FORMATS[dtype],
                                         quant_eps, flags, bool(return_norm))
        if out is None:
            _refused(what)
    return out


def _check_quant(x, group_size, dtype, column_major_scales, scale_ue8m0, quant_eps, what):
    if group_size is not None:
        if group_size <= 0:
            raise ValueError(f"{what}: group_size must be positive")
        if group_size % 1 != 0:
            raise ValueError(f"{what}: group_size must be a whole number")
        if x.ndim >= 1 and x.shape[-1] % group_size != 0:
            raise ValueError(f"{what}: the last dimension of x {x.shape[-1]} must be divisible by group_size {group_size}")
    if column_major_scales and x.ndim != 2:
        raise ValueError(f"{what}: column-major scales need a 2-D input")
    if scale_ue8m0 and dtype == torch.int8:
        raise ValueError(f"{what}: power-of-two scales are for the 8-bit floats")
    if not 0.0 <= quant_eps < _MAX_EPS:
        raise ValueError(f"{what}: quant_eps must be finite in fp32 and not negative")
