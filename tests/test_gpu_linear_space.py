"""fused_linear's backward pass takes memory for its results and for what the wanted ones need, no more."""

import ctypes

import pytest
import torch

import flaggems_vllm_b200 as fg
from flaggems_vllm_b200 import _lib
from test_gpu_linear import make
from test_gpu_norm_balance_bounds import CODE, Guarded, stream

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
M, K, N = 8192, 512, 2048
SLACK = 1 << 20  # the allocator's rounding of a few blocks


def sums(W):
    return 512 * W * 4  # of the bias' gradient: at most 512 rows in fp32


def taken(act, wanted, dtype=BF, bias=False, dy=None, x=None):
    """Bytes at the highest point of a backward pass above what was there before, and the bytes of its results."""
    W = 2 * N if act == "silu_and_mul" else N
    x = torch.randn(M, K, device=DEV).to(dtype) if x is None else x
    w = torch.randn(W, K, device=DEV).to(dtype) / 16
    b = torch.randn(W, device=DEV) if bias else None
    leaves = {"x": x, "w": w, "b": b}
    for n in wanted:
        leaves[n].requires_grad_()
    dy = torch.randn(M, N, device=DEV).to(dtype) if dy is None else dy
    y = fg.fused_linear(x, w, b, act)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    grads = torch.autograd.grad(y, [leaves[n] for n in wanted], dy)
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before, sum(g.numel() * g.element_size() for g in grads)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("wanted", ["x", "w", "xw"])
def test_a_projection_takes_its_results_only(wanted, dtype):
    peak, results = taken(None, wanted, dtype)
    assert peak <= results + SLACK


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_bias_takes_its_sums(dtype):
    peak, results = taken(None, "xwb", dtype, bias=True)
    assert peak <= results + sums(N) + SLACK
    for act, W in (("silu", N), ("silu_and_mul", 2 * N), (None, N)):
        peak, results = taken(act, "b", dtype, bias=True)  # dz is summed as it is formed
        assert peak <= results + sums(W) + SLACK


@pytest.mark.parametrize("dtype", [BF, F32])
def test_an_activation_takes_dz(dtype):
    for act, W in (("gelu", N), ("silu_and_mul", 2 * N)):
        peak, results = taken(act, "xw", dtype)
        assert peak <= results + M * W * dtype.itemsize + SLACK


def test_rows_that_are_copied_take_their_copies():
    odd = torch.randn(M * N + 1, device=DEV).to(BF)[1:].view(M, N)
    peak, results = taken(None, "xw", dy=odd)
    assert peak <= results + M * N * 2 + SLACK
    x = torch.randn(M * K + 1, device=DEV).to(BF)[1:].view(M, K)
    peak, results = taken(None, "xw", x=x)
    assert peak <= results + M * K * 2 + SLACK
    peak, results = taken(None, "x", x=x.detach())  # x is no operand of its own gradient
    assert peak <= results + SLACK


@pytest.mark.parametrize("act,number", [(None, 0), ("gelu", 3), ("silu_and_mul", 5)])
@pytest.mark.parametrize("dtype", [BF, torch.float16, F32])
@pytest.mark.parametrize("rows,cols,n,odd", [(1, 1, 1, 0), (40, 264, 96, 0), (40, 264, 96, 1), (333, 65, 129, 0), (2304, 72, 1032, 1)])
def test_every_set_of_results_in_its_own_space(rows, cols, n, odd, dtype, act, number):
    """Each set of wanted gradients, in exactly the workspace that is said for it, has the bits that all together have."""
    x, w, b, _ = make(rows, cols, n, dtype, act, "f32")
    W, s, c, lib = w.shape[0], dtype.itemsize, CODE[dtype], _lib.lib()
    dy = torch.randn(rows * n + odd, device=DEV).to(dtype)[odd:].view(rows, n)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(fg.fused_linear(*leaves, act), leaves, dy)
    z = torch.zeros(rows, W, dtype=F32 if act == "silu_and_mul" else dtype, device=DEV)
    y, need, status = torch.empty(rows, n, dtype=dtype, device=DEV), ctypes.c_int64(), _lib.status_word(x.device).data_ptr()
    _lib.check(lib.moe_fused_linear_workspace(x.data_ptr(), cols, w.data_ptr(), cols, c, rows, n, cols, number, ctypes.addressof(need)))
    ws = torch.empty(max(need.value, 16), dtype=torch.uint8, device=DEV)
    _lib.check(lib.moe_fused_linear(x.data_ptr(), cols, w.data_ptr(), cols, b.data_ptr(), _lib.MOE_F32, None, n, c, rows, n, cols, number, y.data_ptr(), n,
                                    z.data_ptr(), W, ws.data_ptr(), need.value, status, stream()))
    for mask in range(1, 8):
        dx, dw, db = (bool(mask >> i & 1) for i in range(3))
        _lib.check(lib.moe_fused_linear_grad_workspace_of(dy.data_ptr(), x.data_ptr() if dw else None, cols, w.data_ptr() if dx else None, cols, c, rows, n,
                                                          cols, number, dx, dw, db, ctypes.addressof(need)))
        g = Guarded(0x5A, ws=need.value, dx=rows * cols * s, dw=W * cols * s, db=W * 4)
        _lib.check(lib.moe_fused_linear_grad(dy.data_ptr(), z.data_ptr(), W, x.data_ptr() if dw else None, cols, w.data_ptr() if dx else None, cols, c, rows,
                                             n, cols, number, g.ptr("dx") if dx else None, g.ptr("dw") if dw else None, g.ptr("db") if db else None,
                                             _lib.MOE_F32, g.ptr("ws") if need.value else None, need.value, status, stream()))
        assert g.intact()
        for name, type_, wanted, all_ in (("dx", dtype, dx, want[0]), ("dw", dtype, dw, want[1]), ("db", F32, db, want[2])):
            if wanted:
                assert torch.equal(g.view(name, type_, *all_.shape), all_), (mask, name)
            else:
                assert (g.view(name, torch.uint8, -1) == 0x5A).all()
    assert fg.read_status() == 0
