"""Values of the 8-bit norm and of the gradients where rows lie apart or begin at odd addresses.

The row distance and the addresses choose between pieces of 32 and 16 bytes and single elements, and the groups that a warp
holds between the kernels.  Tolerances are those of test_gpu_norm: counted roundings."""

import pytest
import torch

import flaggems_vllm_b200 as fg
from test_gpu_norm import DEV, EPS, check_grads, check_quant, make, plain

pytestmark = pytest.mark.gpu

LAYOUTS = [(8, 0), (64, 8), (1, 0), (0, 1), (3, 5), (16, 0)]


@pytest.mark.parametrize("gap,offset", LAYOUTS)
@pytest.mark.parametrize("cols,groups", [(512, (None, 256, 128, 64, 32, 8, 2)), (2048, (None, 128)), (7168, (128,)), (1000, (None, 8, 40)),
                                         (8200, (None, 8)), (16400, (None, 16))])
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.int8])
def test_quant(dtype, cols, groups, gap, offset):
    for in_dtype in (torch.bfloat16, torch.float32):
        for M, residual in ((1, True), (37, True), (37, False)):
            x, r, w, _ = make(M, cols, in_dtype, residual, seed=cols + gap, gap=gap, offset=offset)
            want, h, _ = plain(x, w, r)
            for group in groups:
                out = fg.rms_norm_quant(x, w, EPS, r, group_size=group, dtype=dtype, column_major_scales=gap == 8)
                q, s = out[:2]
                assert q.is_contiguous() and s.shape == (M, cols // (group or cols))
                if residual:
                    assert torch.equal(out[2], h)
                check_quant(q, s, want, group or cols, dtype, 1e-10, False, cols)


@pytest.mark.parametrize("gap,offset", LAYOUTS)
@pytest.mark.parametrize("cols", [1, 100, 128, 501, 1023, 1024, 2048, 2056, 4097, 7168, 16384, 33000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradient_of_rows_apart(cols, dtype, gap, offset):
    """Without a residual the backward pass reads x itself, where it lies."""
    for M in (1, 5, 333):
        x, _, w, g = make(M, cols, dtype, False, seed=M + cols, gap=gap, offset=offset)
        dy = torch.randn((M, cols), generator=g, device=DEV).to(dtype)
        xl, wl = x.detach().requires_grad_(), w.clone().requires_grad_()
        dx, dw = torch.autograd.grad(fg.rms_norm(xl, wl, EPS), (xl, wl), dy)
        assert dx.is_contiguous()
        check_grads(x.detach(), None, w, dy, None, dx, dw)


@pytest.mark.parametrize("cols", [100, 1023, 2048, 4097, 16392])
def test_gradient_that_arrives_apart(cols):
    """dy and the stream's gradient as windows, as one row for all, and as columns apart."""
    x, r, w, g = make(40, cols, torch.bfloat16, seed=cols)
    leaves = [t.clone().requires_grad_() for t in (x, w, r)]
    y, h = fg.rms_norm(leaves[0], leaves[1], EPS, leaves[2])
    wide = torch.randn((40, cols + 3), generator=g, device=DEV).bfloat16()
    for dy in (wide[:, 1:cols + 1], wide[:1, :cols].expand(40, cols), wide[:, :cols].t().contiguous().t()):
        for dh in (None, wide[:, 3:], wide[1:2, :cols].expand(40, cols)):
            outs, gs = ([y], [dy]) if dh is None else ([y, h], [dy, dh])
            got = torch.autograd.grad(outs, leaves, gs, retain_graph=True)
            check_grads(x, r, w, dy, dh, got[0], got[1])
            dense = torch.autograd.grad(outs, leaves, [t.contiguous() for t in gs], retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, dense))
