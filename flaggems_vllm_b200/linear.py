"""``fused_linear``: dense product with bias, activation and residual in its epilogue, differentiable.

The products around the routed experts: a shared expert is ``fused_linear(x, w1, activation="silu_and_mul")`` and
``fused_linear(h, w2, residual=routed)`` beside ``fused_experts_impl``; the projections and dense layers between layers of
experts are single calls."""

from __future__ import annotations

import logging
from typing import Optional

import torch

from . import _lib

logger = logging.getLogger(__name__)

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "silu_and_mul": 5}
_MAX_ROWS, _MAX_COLS, _MAX_COLS_F32 = 0x3FFFFFFF, 0x1FFFFFFF, 65535 * 64


def fused_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    activation: Optional[str] = None,
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``, in fp32, rounded once to the type of ``x``.

    ``x`` [..., K], ``weight`` [N, K], ``bias`` [N], ``residual`` and the result [..., N].  ``activation`` is None, "relu",
    "silu", "gelu" (by the normal distribution), "gelu_tanh", or the gated "silu_and_mul": ``weight`` and ``bias`` then have
    2 N rows, gate rows first, and the result is ``silu(z[..., :N]) * z[..., N:]`` (+ residual).

    bfloat16, float16 or float32, one type for ``x``, ``weight`` and ``residual``; ``bias`` may be float32.  Rows may lie in
    wider buffers.  Rows that are no whole number of 16 bytes, or begin at other addresses, are copied first in the 16-bit types.
    Differentiable once, backwards, in all four; where there is an activation, ``x @ weight.T + bias`` is kept for it in the
    type of ``x`` (beyond its largest value as that value), for the gated one in float32.  The gradient of ``x @ weight.T + bias`` is
    rounded to the type of ``x`` in front of the products of the others'; the bias' sums are of its fp32 values.  The same bits in
    every run, whichever gradients are wanted."""
    logger.debug("GEMS FUSED LINEAR")
    act = _ACTIVATIONS.get(activation, -1) if activation is None or isinstance(activation, str) else -1
    if x.is_cuda and act >= 0:
        out = _lib.host().fused_linear(x, weight, bias, act, residual)
        if out is not None:
            return out
    what = "fused_linear"
    if act < 0:
        raise ValueError(f"{what}: activation must be one of {[a for a in _ACTIVATIONS if a]} or None, got {activation!r}")
    _lib.dtype_code(x.dtype)  # ValueError("Unsupported dtype")
    if x.ndim < 1 or weight.ndim != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: x must be [..., K] and weight [N, K], got {list(x.shape)} and {list(weight.shape)}")
    rows, K = weight.shape
    if K == 0 or rows == 0:
        raise ValueError(f"{what}: weight must not be empty")
    if act == 5 and rows % 2 != 0:
        raise ValueError(f"{what}: a gated activation needs an even number of weight rows, got {rows}")
    N = rows // 2 if act == 5 else rows
    if x.numel() // K > _MAX_ROWS or K > _MAX_ROWS or N > _MAX_COLS:
        raise ValueError(f"{what}: at most 2^30 - 1 rows, 2^29 - 1 columns")
    if x.dtype == torch.float32 and max(K, rows) > _MAX_COLS_F32:
        raise ValueError(f"{what}: at most {_MAX_COLS_F32} columns in float32")
    if weight.dtype != x.dtype:
        raise ValueError(f"{what}: weight must be of the type of x, got {weight.dtype}")
    if bias is not None:
        if bias.shape != (rows,):
            raise ValueError(f"{what}: bias must be [{rows}], got {list(bias.shape)}")
        if bias.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{what}: bias must be of the type of x or float32, got {bias.dtype}")
    if residual is not None and (residual.shape != x.shape[:-1] + (N,) or residual.dtype != x.dtype):
        raise ValueError(f"{what}: residual must be {list(x.shape[:-1]) + [N]} of the type of x")
    _lib.require_cuda(x, what)
    for t in (weight, bias, residual):
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: operands on different devices")
    _lib.status_word(x.device)
    out = _lib.host().fused_linear(x, weight, bias, act, residual)  # only the status word was missing
    if out is None:
        out = _lib.host().fused_linear(x.contiguous(), weight.contiguous(), None if bias is None else bias.contiguous(), act,
                                       None if residual is None else residual.contiguous())
    if out is None:
        raise _lib.MoeKernelError(f"{what}: the operands were not taken")
    return out
