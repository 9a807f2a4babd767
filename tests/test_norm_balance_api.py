"""What the norms and the balance loss refuse, before any device work; C entry points with arguments that they reject."""

import ctypes

import pytest
import torch

import flaggems_vllm
import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib


def test_names_are_exported():
    for name in ("rms_norm", "fused_add_rms_norm", "rms_norm_quant", "moe_balance_loss"):
        assert name in fg.__all__ and getattr(flaggems_vllm, name) is getattr(fg, name)


def test_norm_refusals():
    x, w = torch.zeros(4, 64), torch.ones(64)
    for bad, match in ((dict(x=torch.zeros(())), "last dimension"), (dict(x=torch.zeros(4, 0)), "last dimension"),
                       (dict(x=x.double()), "Unsupported dtype"), (dict(x=x.int()), "Unsupported dtype"),
                       (dict(weight=torch.ones(63)), "weight must be"), (dict(weight=torch.ones(1, 64)), "weight must be"),
                       (dict(weight=w.half()), "type of x or float32"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
                       (dict(eps=float("inf")), "eps"), (dict(residual=torch.zeros(4, 63)), "residual"),
                       (dict(residual=torch.zeros(64)), "residual"), (dict(residual=x.half()), "residual")):
        args = {"x": x, "weight": w, **bad}
        with pytest.raises(ValueError, match=match):
            fg.rms_norm(**args)
        with pytest.raises(ValueError, match=match):
            fg.rms_norm_quant(**args)
        if "residual" in bad or "eps" in bad:
            with pytest.raises(ValueError, match=match):
                fg.fused_add_rms_norm(**{"residual": x.clone(), **args})
    with pytest.raises(ValueError, match="there must be a residual"):
        fg.fused_add_rms_norm(x, None, w)
    for call in (lambda: fg.rms_norm(x, w), lambda: fg.rms_norm(x, w, residual=x), lambda: fg.fused_add_rms_norm(x, x, w),
                 lambda: fg.rms_norm_quant(x, w, group_size=32)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_quant_refusals():
    x, w = torch.zeros(4, 64), torch.ones(64)
    with pytest.raises(NotImplementedError, match="8-bit format"):
        fg.rms_norm_quant(x, w, dtype=torch.uint8)
    for bad, match in ((dict(group_size=48), "divisible"), (dict(group_size=0), "positive"), (dict(group_size=-1), "positive"),
                       (dict(scale_ue8m0=True, dtype=torch.int8), "power-of-two"), (dict(quant_eps=-1.0), "quant_eps"),
                       (dict(quant_eps=float("nan")), "quant_eps")):
        with pytest.raises(ValueError, match=match):
            fg.rms_norm_quant(x, w, **bad)
    with pytest.raises(ValueError, match="2-D"):
        fg.rms_norm_quant(x.view(2, 2, 64), w, column_major_scales=True)


def test_balance_refusals():
    l, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for bad, error, match in ((dict(scoring_func="tanh"), ValueError, "scoring_func"), (dict(router_logits=l[0]), ValueError, "tokens"),
                              (dict(topk_ids=ids[:3]), ValueError, "tokens"), (dict(topk_ids=ids.float()), TypeError, "int32"),
                              (dict(router_logits=l.double()), ValueError, "Unsupported dtype"),
                              (dict(router_logits=torch.zeros(4, 1025)), NotImplementedError, "1024"),
                              (dict(router_logits=torch.zeros(4, 0)), NotImplementedError, "1024"),
                              (dict(topk_ids=torch.zeros(4, 33, dtype=torch.int32)), NotImplementedError, "32"),
                              (dict(topk_ids=torch.zeros(4, 0, dtype=torch.int32)), NotImplementedError, "32"),
                              (dict(cu_seqlens=torch.zeros(3)), ValueError, "cu_seqlens"),
                              (dict(cu_seqlens=torch.zeros(1, dtype=torch.int32)), ValueError, "cu_seqlens"),
                              (dict(cu_seqlens=torch.zeros(65537, dtype=torch.int32)), NotImplementedError, "65535"),
                              (dict(is_padding=torch.zeros(4)), ValueError, "is_padding"),
                              (dict(is_padding=torch.zeros(3, dtype=torch.bool)), ValueError, "is_padding")):
        with pytest.raises(error, match=match):
            fg.moe_balance_loss(**{"router_logits": l, "topk_ids": ids, **bad})
    with pytest.raises(RuntimeError, match="no CPU path"):
        fg.moe_balance_loss(l, ids)


def test_c_entry_points_reject_bad_arguments():
    """Host checks only: no call here gets as far as a launch (pointers are never followed)."""
    lib, before = _lib.lib(), _lib.LAUNCHES
    P = 1 << 20  # stands for memory that is 16-byte aligned

    def norm(rows=4, cols=64, dtype=0, wdtype=0, eps=1e-6, x=P, x_ld=64, r=None, w=P, y=2 * P, y_ld=64, h=None, h_ld=64):
        return lib.moe_rms_norm(x, x_ld, r, 64, w, dtype, wdtype, rows, cols, eps, y, y_ld, h, h_ld, None)

    assert norm(rows=0) == 0
    for bad in (dict(rows=-1), dict(cols=0), dict(cols=(1 << 24) + 1), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(w=None),
                dict(y=None), dict(y_ld=63), dict(r=P), dict(r=P, h=P, h_ld=8), dict(x_ld=-1), dict(y=P), dict(r=3 * P, h=2 * P),
                dict(r=3 * P, h=4 * P, y=P, y_ld=72), dict(r=3 * P, h=3 * P, h_ld=72)):
        assert norm(**bad) == -1, bad
    assert norm(rows=1 << 31) == -5
    assert norm(dtype=3) == -2 and norm(dtype=1, wdtype=2) == -2

    def quant(fmt=0, group=32, qeps=1e-10, flags=0, q=P, s=P, s_ld=4, y=None, r=None, r_ld=64, h=None):
        return lib.moe_rms_norm_quant(P, 64, r, r_ld, P, 0, 0, 4, 64, 1e-6, fmt, group, qeps, flags, q, s, s_ld, y, h, None)

    for bad, code in ((dict(fmt=3), -2), (dict(group=0), -3), (dict(group=48), -3), (dict(qeps=-1.0), -1), (dict(flags=2, fmt=2), -1),
                      (dict(q=None), -1), (dict(s=None), -1), (dict(flags=1, s_ld=3), -1), (dict(y=P), -1),
                      (dict(r=2 * P, h=2 * P, r_ld=72), -1), (dict(r=2 * P, h=3 * P, y=3 * P), -1), (dict(r=2 * P, h=3 * P, y=2 * P), -1)):
        assert quant(**bad) == code, bad

    need = ctypes.c_int64()
    assert lib.moe_rms_norm_grad_workspace(4, 0, ctypes.addressof(need)) == -1 and lib.moe_rms_norm_grad_workspace(4, 64, None) == -1
    assert lib.moe_rms_norm_grad_workspace(4, 64, ctypes.addressof(need)) == 0 and need.value == 4 * (4 * 64 + 4)

    def grad(dy=P, dx=P, dw=P, ws=P, size=need.value, rows=4):
        return lib.moe_rms_norm_grad(dy, None, P, 64, P, 0, 0, rows, 64, 1e-6, dx, dw, ws, size, None)

    for bad in (dict(dy=None), dict(dx=None, dw=None), dict(ws=None), dict(size=need.value - 1), dict(ws=P + 4), dict(rows=-1)):
        assert grad(**bad) == -1, bad

    two = (ctypes.c_int64 * 2)()
    assert lib.moe_balance_loss_workspace(100, 16, 2, 1, ctypes.addressof(two)) == 0 and two[1] == 4 * (16 + 1 + 1)
    for bad in ((-1, 16, 2, 1), (4, 0, 2, 1), (4, 16, 0, 1), (4, 16, 2, 0)):
        assert lib.moe_balance_loss_workspace(*bad, ctypes.addressof(two)) == -1
    for bad in ((4, 1025, 2, 1), (4, 16, 33, 1), (4, 16, 2, 65536), (1 << 30, 16, 2, 1)):
        assert lib.moe_balance_loss_workspace(*bad, ctypes.addressof(two)) == -5

    def loss(l=P, dtype=0, ids=P, cu=None, seqs=1, out=P, counts=P, saved=P, ws=P, size=1 << 40):
        return lib.moe_balance_loss(l, 16, dtype, 100, 16, ids, 0, 2, 0, cu, seqs, None, out, counts, saved, ws, size, None, None)

    for bad in (dict(l=None), dict(ids=None), dict(seqs=2), dict(out=None), dict(counts=None), dict(saved=None), dict(ws=None), dict(size=64),
                dict(ws=P + 8)):
        assert loss(**bad) == -1, bad
    assert loss(dtype=3) == -2
    assert lib.moe_balance_loss_grad(None, 16, 0, 100, 16, 2, 0, None, 1, None, P, P, P, None) == -1
    assert _lib.LAUNCHES == before


@pytest.mark.parametrize("tokens", [1, 31, 100, 4097, 65536, 1 << 24])
@pytest.mark.parametrize("experts", [1, 8, 60, 256, 1024])
def test_balance_workspace_covers_every_plan(tokens, experts):
    """The room is that of the plan with most blocks; more sequences need more."""
    one, many = (ctypes.c_int64 * 2)(), (ctypes.c_int64 * 2)()
    _lib.check(_lib.lib().moe_balance_loss_workspace(tokens, experts, 1, 1, ctypes.addressof(one)))
    _lib.check(_lib.lib().moe_balance_loss_workspace(tokens, experts, 1, 1000, ctypes.addressof(many)))
    assert many[0] >= one[0] + 999 * experts * 8 and many[1] == 4 * (1000 * (experts + 1) + 1)
