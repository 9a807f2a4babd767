"""moe_balance_loss: the auxiliary loss that keeps a router's experts evenly used, and the tokens per expert.

It takes what the router had and gave: the logits (``router_gemm``) and the expert ids (``topk_softmax``,
``topk_sigmoid`` or ``grouped_topk``, whose -1 for padded tokens it knows)."""

from __future__ import annotations

import logging
from typing import Optional, Tuple

import torch

from . import _lib

logger = logging.getLogger(__name__)

_MAX_EXPERTS, _MAX_TOPK, _MAX_SEQUENCES, _MAX_ROUTES = 1024, 32, 65535, 0x7FFF0000


def moe_balance_loss(
    router_logits: torch.Tensor,
    topk_ids: torch.Tensor,
    scoring_func: str = "softmax",
    cu_seqlens: Optional[torch.Tensor] = None,
    is_padding: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Returns (loss, counts): a fp32 scalar, and the routes to every expert as int32 [E], or [sequences, E] with
    ``cu_seqlens``.

    Per sequence of N tokens that are not padding, ``loss = sum_e f_e P_e`` with ``f_e = E counts_e / (topk N)`` and
    ``P_e`` the mean over its tokens of the router's score: ``softmax(logits)``, or for ``"sigmoid"`` the sigmoids of the
    row divided by their sum.  1 is even use.  Sequences are the rows ``cu_seqlens[s] : cu_seqlens[s + 1]`` (int32, on the
    device; without it all rows are one); the loss is the mean over those that have a token, 0 if none has.  Rows
    outside them and rows where ``is_padding`` count for nothing, whatever they hold, and get a gradient of zero; a row
    whose logits are all -inf has scores of zero.

    ``topk_ids`` [tokens, topk]: a negative id is no route; one beyond the experts is skipped and reported
    (``read_status``), as are ``cu_seqlens`` that decrease or leave the rows, whose loss is NaN.  Differentiable once in
    the logits, the counts held; the same bits in every run.  At most 1024 experts and 32 routes per token."""
    logger.debug("GEMS MOE BALANCE LOSS")
    if scoring_func not in ("softmax", "sigmoid"):
        raise ValueError(f"scoring_func must be 'softmax' or 'sigmoid', got {scoring_func!r}")
    sigmoid = scoring_func == "sigmoid"
    if router_logits.is_cuda:
        out = _lib.host().balance_loss(router_logits, topk_ids, sigmoid, cu_seqlens, is_padding)
        if out is not None:
            return out
    logits, ids = router_logits, topk_ids
    if logits.ndim != 2 or ids.ndim != 2 or logits.shape[0] != ids.shape[0]:
        raise ValueError("router_logits must be [tokens, experts] and topk_ids [tokens, topk]")
    _lib.dtype_code(logits.dtype)  # ValueError("Unsupported dtype")
    if not 1 <= logits.shape[1] <= _MAX_EXPERTS:
        raise NotImplementedError(f"moe_balance_loss supports 1 to {_MAX_EXPERTS} experts")
    if not 1 <= ids.shape[1] <= _MAX_TOPK:
        raise NotImplementedError(f"moe_balance_loss supports 1 to {_MAX_TOPK} routes per token")
    if ids.dtype not in (torch.int32, torch.int64, torch.uint32):
        raise TypeError("topk_ids must be int32/int64/uint32")
    if ids.numel() > _MAX_ROUTES:
        raise ValueError("moe_balance_loss: at most 2^31 - 2^16 routes")
    if cu_seqlens is not None:
        if cu_seqlens.ndim != 1 or cu_seqlens.dtype != torch.int32 or cu_seqlens.numel() < 2:
            raise ValueError("cu_seqlens must be int32 [sequences + 1] with at least one sequence")
        if cu_seqlens.numel() - 1 > _MAX_SEQUENCES:
            raise NotImplementedError(f"moe_balance_loss supports at most {_MAX_SEQUENCES} sequences")
    if is_padding is not None and (is_padding.dtype != torch.bool or is_padding.shape != (logits.shape[0],)):
        raise ValueError("is_padding must be bool [tokens]")
    _lib.require_cuda(logits, "moe_balance_loss")
    for t in (ids, cu_seqlens, is_padding):
        if t is not None and t.device != logits.device:
            raise ValueError("moe_balance_loss: operands on different devices")
    _lib.status_word(logits.device)
    if ids.dtype == torch.uint32:  # what topk_softmax may write: ids below 2^31, and -1 for padded tokens
        ids = ids.contiguous().view(torch.int32)
    out = _lib.host().balance_loss(logits.contiguous(), ids.contiguous(), sigmoid,
                                   None if cu_seqlens is None else cu_seqlens.contiguous(),
                                   None if is_padding is None else is_padding.contiguous())
    if out is None:
        raise _lib.MoeKernelError("moe_balance_loss: the operands were not taken")
    return out
