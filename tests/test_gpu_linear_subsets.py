"""fused_linear: a gradient has the same bits whichever others are wanted beside it."""

import pytest
import torch

import flaggems_vllm_b200 as fg
from test_gpu_linear import ACTS, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K,N,odd", [(40, 264, 96, 0), (40, 264, 96, 1), (333, 65, 129, 0), (2304, 72, 1032, 1)])
def test_every_set_of_gradients(M, K, N, odd, dtype, act):
    args = make(M, K, N, dtype, act, "f32", True)
    dy = torch.randn(M * N + odd, device=DEV).to(dtype)[odd:].view(M, N)
    want = None
    for mask in range(15, 0, -1):
        ts = [t.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(args)]
        y = fg.fused_linear(ts[0], ts[1], ts[2], act, ts[3])
        y.backward(dy)
        want = [t.grad for t in ts] if want is None else want
        for i in range(4):
            assert (ts[i].grad is None) if not mask >> i & 1 else torch.equal(ts[i].grad, want[i]), (mask, i)
