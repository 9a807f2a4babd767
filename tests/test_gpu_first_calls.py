"""The first call of a thread, and the first ones of a process, made by several threads at once."""

import subprocess
import sys
import threading

import pytest
import torch

import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib, testing

pytestmark = pytest.mark.gpu


def operators():
    x, w = torch.randn(300, 512, device="cuda").bfloat16(), torch.randn(256, 512, device="cuda").bfloat16()
    w1, s1 = testing.make_fp8_block_weights(8, 256, 512, "cuda", seed=1)
    w2, s2 = testing.make_fp8_block_weights(8, 512, 128, "cuda", seed=2)
    v1, v2 = testing.make_half_weights(8, 256, 512, "cuda", seed=1), testing.make_half_weights(8, 512, 128, "cuda", seed=2)
    router, bias = torch.randn(8, 512, device="cuda").bfloat16(), torch.zeros(8, device="cuda")
    weights, ids = torch.full((300, 2), 0.5, device="cuda"), torch.tensor([[1, 6]], device="cuda", dtype=torch.int32).repeat(300, 1)

    def train():
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        y = fg.fused_linear(*leaves, None, "silu")
        return (y.detach(), *torch.autograd.grad(y, leaves, y.detach()))

    return {
        "fused_linear": lambda: (fg.fused_linear(x, w),),
        "fused_linear training": train,
        "fused_linear fp32": lambda: (fg.fused_linear(weights, weights),),
        "few tokens e4m3": lambda: fg.fused_moe_few_tokens(x[:4], router, w1, w2, 2, w1_scale=s1, w2_scale=s2, return_routing=True),
        "few tokens": lambda: fg.fused_moe_few_tokens(x[:4], router, v1, v2, 2, return_routing=True),
        "router": lambda: (fg.router_gemm(x, router),),
        "router and choice": lambda: fg.router_gemm_grouped_topk(x, router, 2, 1, 2, True, 1.0, bias, 1),
        "layer e4m3": lambda: (fg.fused_experts_impl(x, w1, w2, weights, ids, use_fp8_w8a8=True, w1_scale=s1, w2_scale=s2, block_shape=[128, 128]),),
        "layer": lambda: (fg.fused_experts_impl(x, v1, v2, weights, ids),),
        "layer of one token": lambda: (fg.fused_experts_impl(x[:1], v1, v2, weights[:1], ids[:1]),),
    }


def in_threads(run, n):
    """What n new threads get that call it at once."""
    barrier, got, errors = threading.Barrier(n), [], []

    def body():
        barrier.wait()
        try:
            got.append(run())
        except Exception as e:
            errors.append(repr(e))

    threads = [threading.Thread(target=body) for _ in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert len(got) == n
    return got


def test_first_call_of_a_thread():
    """A thread that has not used the device yet; what the calls allocate is there already, so that nothing else uses it for them."""
    for name, run in operators().items():
        want = run()
        torch.cuda.synchronize()
        (got,) = in_threads(run, 1)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
    assert fg.read_status() == 0


def first_calls(name):
    run = operators()[name]
    _lib.host()
    _lib.status_word("cuda")
    torch.cuda.synchronize()
    sys.setswitchinterval(1e-6)
    got = in_threads(run, 12)
    want = run()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want)) and fg.read_status() == 0


@pytest.mark.parametrize("name", ["fused_linear", "few tokens e4m3"])
def test_first_calls_of_a_process(name):
    program = f"import sys; sys.path[:0] = ['tests', '.']; import test_gpu_first_calls as t; t.first_calls({name!r})"
    r = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
