"""A shared expert in e4m3 for any number of tokens: the layer of one expert beside the routed ones, as it is for few tokens in one call."""

import pytest
import torch

import flaggems_vllm_b200 as fg
from test_gpu_few_tokens import call, make

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def layers(d, tw, ti):
    """Routed experts, shared expert and residual, one behind another."""
    x, M = d["x"], d["x"].shape[0]
    fp8 = dict(use_fp8_w8a8=True, block_shape=[128, 128])
    routed = fg.fused_experts_impl(x, d["w1"], d["w2"], tw, ti, w1_scale=d["w1_scale"], w2_scale=d["w2_scale"], **fp8)
    one, first = torch.ones(M, 1, device="cuda"), torch.zeros(M, 1, device="cuda", dtype=torch.int32)
    shared = fg.fused_experts_impl(x, d["shared_w1"][None], d["shared_w2"][None], one, first, w1_scale=d["shared_w1_scale"][None],
                                   w2_scale=d["shared_w2_scale"][None], **fp8)
    return routed, shared, routed + shared + d["residual"]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M", [1, 3, 8])
def test_one_call_and_layers(M, dtype):
    d = make(M, 32, 1024, 512, 768, dtype, fp8=True, residual=True)
    out, tw, ti = call(d, 6, "sigmoid", 4, 2, 2.5)
    want = layers(d, tw, ti)[2]
    assert (out.double() - want.double()).norm() <= 1e-2 * want.double().norm()


@pytest.mark.parametrize("M", [9, 300])
def test_more_tokens_are_each_ones_own(M):
    """Tokens of a prompt beside the same tokens eight at a time."""
    d = make(M, 32, 1024, 512, 768, BF, fp8=True, residual=True)
    scores = fg.router_gemm(d["x"], d["router"]).sigmoid()
    tw, ti = fg.grouped_topk(scores, 4, 2, 6, True, 2.5, d["bias"], 0)
    want = layers(d, tw, ti)[2]
    for at in range(0, M, 8):
        few = dict(d, x=d["x"][at:at + 8], residual=d["residual"][at:at + 8])
        out, _, ids = call(few, 6, "sigmoid", 4, 2, 2.5)
        same = (ids == ti[at:at + 8]).all(1)  # a near tie may be decided otherwise in other bits of the logits
        assert same.float().mean() >= 0.75
        part = want[at:at + 8][same].double()
        assert (out[same].double() - part).norm() <= 1e-2 * part.norm()
