"""What fused_linear and fused_moe_few_tokens refuse, before any device work; C entry points with arguments that they reject."""

import ctypes
import os
import re

import pytest
import torch

import flaggems_vllm
import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib


def test_names_are_exported():
    for name in ("fused_linear", "fused_moe_few_tokens"):
        assert name in fg.__all__ and getattr(flaggems_vllm, name) is getattr(fg, name)


def test_linear_refusals():
    x, w = torch.zeros(4, 64), torch.ones(32, 64)
    for bad, match in ((dict(x=torch.zeros(())), "must be"), (dict(x=torch.zeros(4, 63)), "must be"), (dict(weight=torch.ones(64)), "must be"),
                       (dict(weight=torch.ones(1, 32, 64)), "must be"), (dict(x=torch.zeros(4, 0), weight=torch.ones(32, 0)), "empty"),
                       (dict(weight=torch.ones(0, 64)), "empty"), (dict(x=x.double()), "Unsupported dtype"), (dict(x=x.int()), "Unsupported dtype"),
                       (dict(weight=w.half()), "type of x"), (dict(x=x.half()), "type of x"), (dict(bias=torch.zeros(33)), "bias must be"),
                       (dict(bias=torch.zeros(1, 32)), "bias must be"), (dict(bias=torch.zeros(32).half()), "bias must be"),
                       (dict(residual=torch.zeros(4, 31)), "residual"), (dict(residual=torch.zeros(32)), "residual"),
                       (dict(residual=torch.zeros(4, 32).half()), "residual"), (dict(activation="tanh"), "activation"),
                       (dict(activation=""), "activation"), (dict(activation=1), "activation"), (dict(activation=["relu"]), "activation"),
                       (dict(weight=torch.ones(31, 64), activation="silu_and_mul"), "even"),
                       (dict(activation="silu_and_mul", residual=torch.zeros(4, 32)), "residual"),
                       (dict(activation="silu_and_mul", bias=torch.zeros(16)), "bias must be")):
        with pytest.raises(ValueError, match=match):
            fg.fused_linear(**{"x": x, "weight": w, **bad})
    for act in (None, "relu", "silu", "gelu", "gelu_tanh", "silu_and_mul"):
        with pytest.raises(RuntimeError, match="no CPU path"):
            fg.fused_linear(x, w, torch.zeros(32), act)
        with pytest.raises(RuntimeError, match="no CPU path"):
            fg.fused_linear(x.to("meta"), w.to("meta"), None, act)
    with pytest.raises(ValueError, match="2\\^30"):
        fg.fused_linear(torch.zeros(1, 64).expand(1 << 30, 64), w)
    with pytest.raises(ValueError, match="2\\^30"):
        fg.fused_linear(x[:, :1], torch.ones(1, 1).expand(1 << 29, 1))
    for w in (torch.ones(1, 1).expand(4194241, 1), torch.ones(1, 1).expand(1, 4194241)):
        with pytest.raises(ValueError, match="4194240 columns in float32"):
            fg.fused_linear(torch.zeros(1, 1).expand(2, w.shape[1]), w)


def layer(dtype=torch.bfloat16, M=2, E=8, H=128, I=128, shared=0, fp8=False):
    held = torch.float8_e4m3fn if fp8 else dtype
    d = dict(hidden_states=torch.zeros(M, H, dtype=dtype), router_weight=torch.zeros(E, H, dtype=dtype),
             w1=torch.zeros(E, 2 * I, H).to(held), w2=torch.zeros(E, H, I).to(held), topk=2)
    if fp8:
        d |= dict(w1_scale=torch.ones(E, 2 * I // 128, H // 128), w2_scale=torch.ones(E, H // 128, I // 128))
    if shared:
        d |= dict(shared_w1=torch.zeros(2 * shared, H).to(held), shared_w2=torch.zeros(H, shared).to(held))
        if fp8:
            d |= dict(shared_w1_scale=torch.ones(2 * shared // 128, H // 128), shared_w2_scale=torch.ones(H // 128, shared // 128))
    return d


def test_few_tokens_refusals():
    z = torch.zeros
    bf = torch.bfloat16
    for bad, match in ((dict(scoring="tanh"), "scoring"), (dict(scoring=None), "scoring"), (dict(hidden_states=z(2, 128)), "Unsupported dtype"),
                       (dict(hidden_states=z(2, 128, dtype=torch.float64)), "Unsupported dtype"), (dict(hidden_states=z(128, dtype=bf)), "must be"),
                       (dict(hidden_states=z(1, 2, 128, dtype=bf)), "must be"), (dict(hidden_states=z(9, 128, dtype=bf)), "at most 8 tokens"),
                       (dict(hidden_states=z(2, 192, dtype=bf)), "belong together"), (dict(router_weight=z(7, 128, dtype=bf)), "belong together"),
                       (dict(router_weight=z(8, 128, dtype=torch.half)), "router_weight"), (dict(w1=z(8, 255, 128, dtype=bf)), "belong together"),
                       (dict(w2=z(8, 128, 64, dtype=bf)), "belong together"), (dict(w1=z(8, 256, 128)), "w1 must be"),
                       (dict(w2=z(8, 128, 128, dtype=torch.half)), "w2 must be"), (dict(topk=0), "topk"), (dict(topk=9), "topk"), (dict(topk=-1), "topk"),
                       (dict(num_expert_group=3), "groups"), (dict(num_expert_group=0), "groups"), (dict(num_expert_group=4, topk_group=5), "groups"),
                       (dict(num_expert_group=4, topk_group=0), "groups"), (dict(num_expert_group=4, topk_group=1, topk=3), "topk"),
                       (dict(routed_scaling_factor=float("nan")), "finite"), (dict(routed_scaling_factor=float("inf")), "finite"),
                       (dict(routed_scaling_factor=1e39), "finite"), (dict(e_score_correction_bias=z(7)), "e_score_correction_bias"),
                       (dict(e_score_correction_bias=z(8, dtype=torch.int32)), "e_score_correction_bias"), (dict(residual=z(2, 128)), "residual"),
                       (dict(residual=z(1, 128, dtype=bf)), "residual"), (dict(shared_w1=z(128, 128, dtype=bf)), "come together"),
                       (dict(shared_w1=z(128, 128, dtype=bf), shared_w2=z(128, 128, dtype=bf)), "shared_w1 must be"),
                       (dict(shared_w1=z(128, 128), shared_w2=z(128, 64)), "shared_w1 must be"),
                       (dict(shared_w1=z(0, 128, dtype=bf), shared_w2=z(128, 0, dtype=bf)), "shared_w1 must be"),
                       (dict(shared_w1=z(160, 128, dtype=bf), shared_w2=z(128, 80, dtype=bf)), "multiples of 64"),
                       (dict(w1_scale=z(8, 2, 1)), "w1_scale"), (dict(w2_scale=z(8, 1, 1)), "w2_scale"), (dict(shared_w1_scale=z(1, 1)), "shared_w1_scale")):
        with pytest.raises(ValueError, match=match):
            fg.fused_moe_few_tokens(**{**layer(), **bad})
    for sizes, match in ((dict(H=96), "multiples of 64"), (dict(I=96), "multiples of 64"), (dict(fp8=True, H=192), "multiples of 128"),
                         (dict(fp8=True, shared=64, I=256), "multiples of 128|shared_w1_scale"), (dict(E=1025, H=64, I=64), "1024 experts"),
                         (dict(H=16448, I=64, E=2), "hidden sizes"), (dict(H=8320, E=2, fp8=True), "hidden sizes"),
                         (dict(E=0), "experts")):
        with pytest.raises(ValueError, match=match):
            fg.fused_moe_few_tokens(**layer(**sizes))
    with pytest.raises(ValueError, match="topk"):
        fg.fused_moe_few_tokens(**{**layer(E=64, H=64, I=64), "topk": 33})
    for missing in ("w1_scale", "w2_scale", "shared_w1_scale", "shared_w2_scale"):
        with pytest.raises(ValueError, match=missing):
            fg.fused_moe_few_tokens(**{**layer(fp8=True, shared=128), missing: None})
        with pytest.raises(ValueError, match=missing):
            full = layer(fp8=True, shared=128)
            fg.fused_moe_few_tokens(**{**full, missing: full[missing].half()})
    for leaf in ("hidden_states", "router_weight", "w1", "w2", "shared_w1", "shared_w2", "residual"):
        d = {**layer(shared=64), "residual": torch.zeros(2, 128, dtype=bf)}
        d[leaf] = d[leaf].requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            fg.fused_moe_few_tokens(**d)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            fg.fused_moe_few_tokens(**d)
    for d in (layer(), layer(torch.half, shared=64), layer(fp8=True, shared=128), layer(M=0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            fg.fused_moe_few_tokens(**d)


def test_linear_c_entry_points_reject_bad_arguments():
    """Host checks only: no call here gets as far as a launch (pointers are never followed)."""
    lib, before, P = _lib.lib(), _lib.LAUNCHES, 1 << 20
    need = ctypes.c_int64()
    at = ctypes.addressof(need)

    def space(x=P, x_ld=64, w=P, w_ld=64, dtype=_lib.MOE_BF16, M=4, N=32, K=64, act=0, out=at):
        return lib.moe_fused_linear_workspace(x, x_ld, w, w_ld, dtype, M, N, K, act, out)

    assert space() == 0 and need.value == 0
    assert space(x=P + 2) == 0 and need.value == 512 and space(w_ld=65) == 0 and need.value == 32 * 64 * 2
    assert space(w=P + 8, act=5) == 0 and need.value == 64 * 64 * 2 and space(x=P + 2, dtype=_lib.MOE_F32) == 0 and need.value == 0
    extents = [(dict(M=-1), -1), (dict(N=0), -1), (dict(K=0), -1), (dict(act=6), -1), (dict(act=-1), -1), (dict(dtype=3), -2), (dict(M=1 << 30), -5),
               (dict(N=1 << 29), -5), (dict(K=1 << 30), -5)]
    for bad, code in extents + [(dict(out=None), -1)]:
        assert space(**bad) == code, bad

    def product(x=P, x_ld=64, w=P, w_ld=64, b=None, b_dtype=_lib.MOE_BF16, r=None, r_ld=32, dtype=_lib.MOE_BF16, M=4, N=32, K=64, act=0, y=2 * P,
                y_ld=32, z=None, z_ld=64, ws=None, size=0):
        return lib.moe_fused_linear(x, x_ld, w, w_ld, b, b_dtype, r, r_ld, dtype, M, N, K, act, y, y_ld, z, z_ld, ws, size, None, None)

    assert product(M=0) == 0
    for bad, code in extents + [(dict(x=None), -1), (dict(w=None), -1), (dict(y=None), -1), (dict(b=P, b_dtype=_lib.MOE_F16), -2), (dict(x_ld=63), -3),
                                (dict(w_ld=0), -3), (dict(y_ld=31), -3), (dict(r=P, r_ld=31), -3), (dict(z=P, z_ld=31), -3),
                                (dict(z=P, z_ld=63, act=5), -3), (dict(x=P + 2), -1), (dict(x_ld=65), -1), (dict(x=P + 2, ws=P, size=511), -1),
                                (dict(x=P + 2, ws=P + 8, size=512), -1)]:
        assert product(**bad) == code, bad

    def grad_space(M=4, act=0, dtype=_lib.MOE_BF16, out=at):
        return lib.moe_fused_linear_grad_workspace(P, 64, P, 64, dtype, M, 32, 64, act, out)

    assert grad_space() == 0 and grad_space(out=None) == -1 and grad_space(act=6) == -1 and grad_space(M=-1) == -1

    def grad(dy=P, z=P, z_ld=32, x=P, x_ld=64, w=P, w_ld=64, dtype=_lib.MOE_BF16, M=4, N=32, K=64, act=1, dx=P, dw=P, db=P, db_dtype=_lib.MOE_F32, ws=P,
             size=1 << 20):
        return lib.moe_fused_linear_grad(dy, z, z_ld, x, x_ld, w, w_ld, dtype, M, N, K, act, dx, dw, db, db_dtype, ws, size, None, None)

    for bad, code in extents + [(dict(M=0), -1), (dict(dy=None), -1), (dict(z=None), -1), (dict(x=None), -1), (dict(w=None), -1), (dict(db_dtype=_lib.MOE_F16), -2),
                                (dict(x_ld=63), -3), (dict(w_ld=63), -3), (dict(z_ld=31), -3), (dict(ws=None), -1), (dict(ws=P + 8), -1), (dict(size=255), -1),
                                (dict(size=256), -1)]:
        assert grad(**bad) == code, bad
    assert _lib.LAUNCHES == before


def test_few_tokens_c_entry_points_reject_bad_arguments():
    lib, before, P = _lib.lib(), _lib.LAUNCHES, 1 << 20
    need = ctypes.c_int64()
    at = ctypes.addressof(need)
    assert lib.moe_few_tokens_workspace(4, 8, 128, 0, 2, 0, at) == 0 and need.value > 0
    for bad in ((9, 8, 128, 0, 2, 0, at), (-1, 8, 128, 0, 2, 0, at), (4, 0, 128, 0, 2, 0, at), (4, 1025, 128, 0, 2, 0, at), (4, 8, 0, 0, 2, 0, at),
                (4, 8, 128, -1, 2, 0, at), (4, 8, 128, 0, 0, 0, at), (4, 8, 128, 0, 33, 0, at), (4, 8, 128, 0, 2, 0, None)):
        assert lib.moe_few_tokens_workspace(*bad) == -1, bad

    def few(x=P, x_ld=128, dtype=_lib.MOE_BF16, router=P, r_dtype=_lib.MOE_BF16, w1=P, w2=P, s1=None, s2=None, sw1=None, sw2=None, ss1=None, ss2=None,
            res=None, res_ld=128, M=4, E=8, H=128, I=128, Is=0, topk=2, groups=1, kept=1, out=P, tw=P, ti=P, ws=P, size=1 << 30):
        return lib.moe_few_tokens(x, x_ld, dtype, router, r_dtype, None, w1, w2, s1, s2, sw1, sw2, ss1, ss2, res, res_ld, M, E, H, I, Is, topk, groups, kept,
                                  1, 1.0, 0, out, tw, ti, ws, size, None, None)

    assert few(M=0) == 0
    for bad, code in ((dict(dtype=_lib.MOE_F32), -2), (dict(r_dtype=_lib.MOE_F16), -2), (dict(M=9), -5), (dict(M=-1), -5), (dict(E=0), -3), (dict(E=1025), -3),
                      (dict(H=96), -3), (dict(H=0), -3), (dict(H=16448, x_ld=16448), -3), (dict(I=0), -3), (dict(I=100), -3), (dict(I=(1 << 22) + 64), -3),
                      (dict(Is=32), -3), (dict(Is=-64), -3), (dict(s1=P, s2=P, I=64), -3), (dict(s1=P, s2=P, H=8320, x_ld=8320), -3), (dict(topk=0), -3),
                      (dict(topk=9), -3), (dict(topk=33, E=64), -3), (dict(groups=3), -3), (dict(groups=33, E=66), -3), (dict(kept=2), -3), (dict(kept=0), -3),
                      (dict(groups=4, kept=1, topk=3), -3), (dict(x=None), -1), (dict(router=None), -1), (dict(w1=None), -1), (dict(w2=None), -1),
                      (dict(out=None), -1), (dict(tw=None), -1), (dict(ti=None), -1), (dict(ws=None), -1), (dict(size=need.value - 1), -1),
                      (dict(s1=P), -1), (dict(s2=P), -1), (dict(Is=64), -1), (dict(sw1=P), -1), (dict(Is=64, sw1=P), -1),
                      (dict(s1=P, s2=P, Is=128, sw1=P, sw2=P, ss1=P), -1), (dict(x_ld=127), -3), (dict(x_ld=132), -3), (dict(res=P, res_ld=127), -3),
                      (dict(w1=P + 16), -1), (dict(w2=P + 16), -1), (dict(Is=64, sw1=P + 16, sw2=P), -1), (dict(x=P + 8), -1), (dict(router=P + 8), -1),
                      (dict(ws=P + 8), -1)):
        assert few(**bad) == code, bad
    assert _lib.LAUNCHES == before


@pytest.mark.parametrize("name", ["linear.cu", "few_tokens.cu", "few_tokens_fp8.cu"])
def test_inputs_of_kernels_that_start_early_are_not_read_only(name):
    """A kernel launched before its predecessor has ended may not declare what that one writes constant for its own life."""
    with open(os.path.join(os.path.dirname(flaggems_vllm.__file__), "..", "flaggems_vllm_b200", "csrc", name)) as fh:
        source = fh.read()
    assert "pdl_wait" in source and not re.search(r"const\s+\w+\s*\*\s*__restrict__|__ldg\(|ld\.global\.nc", source)
