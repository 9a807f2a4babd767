"""fused_moe_few_tokens chooses among equal scores as grouped_topk does: the lowest expert, the lowest group."""

import pytest
import torch

import flaggems_vllm_b200 as fg
from test_gpu_few_tokens import call, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
CONFIGS = [(60, 3, 2, 5), (60, 1, 1, 9), (100, 4, 2, 8), (100, 20, 7, 16), (300, 1, 1, 7), (300, 30, 4, 32), (256, 8, 4, 8), (32, 32, 5, 5), (1000, 8, 1, 32),
           (1000, 25, 6, 20), (64, 2, 1, 32)]


@pytest.mark.parametrize("E,groups,kept,topk", CONFIGS)
@pytest.mark.parametrize("M", [1, 4, 8])
@pytest.mark.parametrize("distinct", [1, 2, 5])  # values of the bias
def test_equal_scores_of_all_experts(E, groups, kept, topk, M, distinct):
    """Router rows that are all the same: what is ranked are the bias' few values."""
    d = make(M, E, 128, 64)
    d["router"] = d["router"][:1].repeat(E, 1)
    g = torch.Generator(device=DEV).manual_seed(E + distinct)
    d["bias"] = torch.randint(0, distinct, (E,), generator=g, device=DEV).float() / 8
    _, tw, ti = call(d, topk, "sigmoid", groups, kept, 1.5)
    scores = fg.router_gemm(d["x"], d["router"]).sigmoid()
    assert (scores == scores[:, :1]).all()
    w, i = fg.grouped_topk(scores, groups, kept, topk, True, 1.5, d["bias"], 0)
    assert torch.equal(ti, i)
    torch.testing.assert_close(tw, w, rtol=1e-6, atol=0)
    _, _, ti = call(d, topk, "softmax", groups, kept, 1.5)  # scores of 1 / E, the same ranks
    w, i = fg.grouped_topk(torch.full((M, E), 1 / E, device=DEV), groups, kept, topk, True, 1.5, d["bias"], 0)
    assert torch.equal(ti, i)


@pytest.mark.parametrize("E,groups,kept,topk", CONFIGS)
@pytest.mark.parametrize("M", [1, 2, 4])  # the logits of more tokens have other bits
def test_equal_scores_of_some_experts(E, groups, kept, topk, M):
    """Seven different router rows over and over: experts and whole groups tie."""
    d = make(M, E, 256, 64, bias=False)
    d["router"] = d["router"][torch.arange(E, device=DEV) % 7]
    bias = torch.zeros(E, device=DEV)
    w, i = fg.router_gemm_grouped_topk(d["x"], d["router"], groups, kept, topk, True, 2.5, bias, 1)
    for d["bias"] in (None, bias):
        _, tw, ti = call(d, topk, "sigmoid", groups, kept, 2.5)
        assert torch.equal(ti, i)
        torch.testing.assert_close(tw, w, rtol=1e-6, atol=0)
