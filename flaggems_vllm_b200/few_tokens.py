"""``fused_moe_few_tokens``: router, routed experts, shared expert and residual of one layer, for the tokens of a decode step or of a
speculative draft, in two launches."""

from __future__ import annotations

import logging
import operator
from typing import Optional, Tuple, Union

import torch

from . import _lib

logger = logging.getLogger(__name__)

MAX_FEW_TOKENS = 8
_MAX_EXPERTS, _MAX_TOPK, _MAX_GROUPS, _MAX_WIDTH = 1024, 32, 32, 1 << 22
_MAX_HIDDEN, _MAX_HIDDEN_FP8 = 16384, 8192


def fused_moe_few_tokens(
    hidden_states: torch.Tensor,
    router_weight: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    topk: int,
    renormalize: bool = True,
    scoring: str = "softmax",
    num_expert_group: int = 1,
    topk_group: int = 1,
    routed_scaling_factor: float = 1.0,
    e_score_correction_bias: Optional[torch.Tensor] = None,
    w1_scale: Optional[torch.Tensor] = None,
    w2_scale: Optional[torch.Tensor] = None,
    shared_w1: Optional[torch.Tensor] = None,
    shared_w2: Optional[torch.Tensor] = None,
    shared_w1_scale: Optional[torch.Tensor] = None,
    shared_w2_scale: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    return_routing: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]:
    """``sum_j weight_j * expert_j(x) [+ shared(x)] [+ residual]`` for up to ``MAX_FEW_TOKENS`` tokens, rounded once; with
    ``return_routing`` (out, topk_weights fp32, topk_ids int32).

    ``hidden_states`` [M, H] bfloat16 or float16; ``router_weight`` [E, H] of the same type or float32.  Logits, scores
    (``scoring``: "softmax" or "sigmoid") and the choice among ``score + e_score_correction_bias`` within the ``topk_group``
    best of ``num_expert_group`` groups are those of ``router_gemm`` and ``grouped_topk``, in fp32 (up to four tokens bit for bit): a
    group ranks by the sum of its two best, in either scoring, and of equal experts or groups the lower index comes first.  Weights are
    the scores, divided by their sum where ``renormalize``, times ``routed_scaling_factor``.

    ``w1`` [E, 2 I, H] (gate rows first), ``w2`` [E, H, I] as ``fused_experts_impl`` has them, in the type of the activations, or
    float8_e4m3fn with ``w1_scale`` [E, 2 I / 128, H / 128] and ``w2_scale`` [E, H / 128, I / 128]: the activations are then taken in
    e4m3 too, in groups of 128, as with ``use_fp8_w8a8`` and ``block_shape=[128, 128]``.  The shared expert, [2 Is, H] and [H, Is],
    has the format of the others.  Each expert's intermediate is rounded to the activations' type, as ``fused_experts_impl`` rounds it.
    H (at most 16384, in 8 bits 8192), I and Is are multiples of 64, in 8 bits of 128; at most 1024 experts, 32 per token.

    More tokens: ``router_gemm_grouped_topk``, ``fused_experts_impl`` and, for the shared expert, ``fused_linear`` or in 8 bits a layer
    of one expert.  Not differentiable: refused where a gradient is wanted.  The same bits in every run of the same call; what the other
    tokens of a call choose may change the order of a token's sums."""
    logger.debug("GEMS FUSED MOE FEW TOKENS")
    what = "fused_moe_few_tokens"
    sigmoid = scoring == "sigmoid"
    if not sigmoid and scoring != "softmax":
        raise ValueError(f"{what}: scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    x = hidden_states
    out = None
    if x.is_cuda:
        out = _lib.host().few_tokens(x, router_weight, w1, w2, topk, renormalize, sigmoid, num_expert_group, topk_group,
                                     routed_scaling_factor, e_score_correction_bias, w1_scale, w2_scale, shared_w1, shared_w2,
                                     shared_w1_scale, shared_w2_scale, residual)
    if out is None:
        out = _slow(x, router_weight, w1, w2, topk, renormalize, sigmoid, num_expert_group, topk_group, routed_scaling_factor,
                    e_score_correction_bias, w1_scale, w2_scale, shared_w1, shared_w2, shared_w1_scale, shared_w2_scale, residual, what)
    return out if return_routing else out[0]


def _slow(x, router, w1, w2, topk, renormalize, sigmoid, groups, kept, factor, bias, s1, s2, sw1, sw2, ss1, ss2, residual, what):
    """The checks, and operands brought into the layout that the library takes."""
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"Unsupported dtype: {x.dtype}")
    if x.ndim != 2 or router.ndim != 2 or w1.ndim != 3 or w2.ndim != 3:
        raise ValueError(f"{what}: hidden_states must be [M, H], router_weight [E, H], w1 [E, 2 I, H], w2 [E, H, I]")
    M, H = x.shape
    E, I = router.shape[0], w2.shape[2]
    if M > MAX_FEW_TOKENS:
        raise ValueError(f"{what}: at most {MAX_FEW_TOKENS} tokens, got {M}; more go through router_gemm_grouped_topk and fused_experts_impl")
    if router.shape != (E, H) or w1.shape != (E, 2 * I, H) or w2.shape != (E, H, I):
        raise ValueError(f"{what}: shapes of hidden_states {list(x.shape)}, router_weight {list(router.shape)}, w1 {list(w1.shape)} and "
                         f"w2 {list(w2.shape)} do not belong together")
    if router.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{what}: router_weight must be of the type of hidden_states or float32, got {router.dtype}")
    fp8 = w1.dtype == torch.float8_e4m3fn
    most = _MAX_HIDDEN_FP8 if fp8 else _MAX_HIDDEN
    if not 1 <= E <= _MAX_EXPERTS or not 1 <= I <= _MAX_WIDTH or not 1 <= H <= most:
        raise ValueError(f"{what}: 1 to {_MAX_EXPERTS} experts of 1 to {_MAX_WIDTH} columns, and hidden sizes up to {most}")
    topk, groups, kept = operator.index(topk), operator.index(groups), operator.index(kept)
    if not 1 <= groups <= _MAX_GROUPS or E % groups != 0 or not 1 <= kept <= groups:
        raise ValueError(f"{what}: {groups} groups, {kept} of them kept, do not divide {E} experts")
    if not 1 <= topk <= min(_MAX_TOPK, E // groups * kept):
        raise ValueError(f"{what}: topk must be 1 to {min(_MAX_TOPK, E // groups * kept)}, got {topk}")
    if not abs(float(factor)) < 3e38:
        raise ValueError(f"{what}: routed_scaling_factor must be finite in fp32")
    if (sw1 is None) != (sw2 is None):
        raise ValueError(f"{what}: shared_w1 and shared_w2 come together")
    Is = 0
    if sw1 is not None:
        if sw2.ndim != 2 or sw1.shape != (2 * sw2.shape[1], H) or sw2.shape[0] != H or sw2.shape[1] == 0:
            raise ValueError(f"{what}: shared_w1 must be [2 Is, {H}] and shared_w2 [{H}, Is]")
        Is = sw2.shape[1]
        if Is > _MAX_WIDTH:
            raise ValueError(f"{what}: a shared expert of at most {_MAX_WIDTH} columns")
    held = torch.float8_e4m3fn if fp8 else x.dtype
    for t, n in ((w1, "w1"), (w2, "w2"), (sw1, "shared_w1"), (sw2, "shared_w2")):
        if t is not None and t.dtype != held:
            raise ValueError(f"{what}: {n} must be {held}, got {t.dtype}")
    unit = 128 if fp8 else 64
    if H % unit or I % unit or Is % unit:
        raise ValueError(f"{what}: sizes must be multiples of {unit}, got H {H}, I {I}" + (f", shared {Is}" if Is else ""))
    scales = [(s1, (E, 2 * I // 128, H // 128), "w1_scale", True), (s2, (E, H // 128, I // 128), "w2_scale", True),
              (ss1, (2 * Is // 128, H // 128), "shared_w1_scale", Is > 0), (ss2, (H // 128, Is // 128), "shared_w2_scale", Is > 0)]
    for t, shape, n, needed in scales:
        if (t is not None) != (fp8 and needed):
            raise ValueError(f"{what}: {n} belongs to weights in float8_e4m3fn, and they to it")
        if t is not None and (t.shape != shape or t.dtype != torch.float32):
            raise ValueError(f"{what}: {n} must be float32 {list(shape)}")
    if bias is not None and (bias.numel() != E or not bias.dtype.is_floating_point):
        raise ValueError(f"{what}: e_score_correction_bias must have {E} elements")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{what}: residual must have the shape and type of hidden_states")
    operands = [x, router, w1, w2, bias, s1, s2, sw1, sw2, ss1, ss2, residual]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        raise RuntimeError(f"{what} has no gradient: use fused_linear and the operators of the layer, or torch.no_grad()")
    _lib.require_cuda(x, what)
    if any(t is not None and t.device != x.device for t in operands):
        raise ValueError(f"{what}: operands on different devices")
    if M == 0:
        return (torch.empty_like(x, memory_format=torch.contiguous_format), torch.empty((0, topk), dtype=torch.float32, device=x.device),
                torch.empty((0, topk), dtype=torch.int32, device=x.device))
    _lib.status_word(x.device)

    def laid(t, align):
        """Contiguous, and begun where 16- or 32-byte loads can begin."""
        if t is None:
            return None
        t = t.contiguous()
        return t if t.data_ptr() % align == 0 else t.clone()

    if bias is not None:
        bias = bias.flatten().float().contiguous()
    out = _lib.host().few_tokens(laid(x, 16), laid(router, 16), laid(w1, 32), laid(w2, 32), topk, bool(renormalize), sigmoid, groups, kept,
                                 float(factor), bias, laid(s1, 4), laid(s2, 4), laid(sw1, 32), laid(sw2, 32), laid(ss1, 4), laid(ss2, 4),
                                 laid(residual, 2))
    if out is None:
        raise _lib.MoeKernelError(f"{what}: the operands were not taken")
    return out
