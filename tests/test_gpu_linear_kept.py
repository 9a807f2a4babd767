"""fused_linear: the pre-activation z that is kept in 16 bits for the backward pass still has the slope of the fp32 sum.

z is held to 64 bits exactly where it comes out of the bias alone or far from every step of the slope: dz is then dy times 0 or 1, with no
rounding, and what remains is the products' sums: (n + 2) 2^-23 of the sum of absolute products, one rounding, and half of the
smallest subnormal of f16."""

import pytest
import torch

import flaggems_vllm_b200 as fg

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16
TINY = {HF: 2.0**-25, BF: 2.0**-134}
# tiles with K over a cluster, tiles by pairs, and both with rows that are no whole 16-byte pieces
SIZES = [(3, 72, 48), (40, 264, 1025), (2304, 64, 1024), (2100, 64, 1025)]


def step(dtype, M, K, N, act, bias, slope, w_std):
    """One training step whose slope is `slope` [N] (0 or 1); everything compared."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w, dy = torch.randn(M, K, generator=g, device=DEV).to(dtype), (w_std * torch.randn(N, K, generator=g, device=DEV)).to(dtype), \
        torch.randn(M, N, generator=g, device=DEV).to(dtype)
    leaves = [t.requires_grad_() for t in (x, w, bias.clone())]
    y = fg.fused_linear(*leaves, act)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    dz = dy.double() * slope.double()
    X, W, u = x.detach().double(), w.detach().double(), torch.finfo(dtype).eps / 2
    for name, got, a, b, n in (("dx", dx, dz, W, N), ("dw", dw, dz.t(), X, M)):
        want, off = a @ b, (n + 2) * 2.0**-23 * (a.abs() @ b.abs())
        assert got.isfinite().all(), name
        assert ((got.double() - want).abs() <= off + u * (want.abs() + off) + TINY[dtype]).all(), name
    assert db.dtype == torch.float32 and db.isfinite().all()
    assert ((db.double() - dz.sum(0)).abs() <= (M + 16) * 2.0**-23 * dz.abs().sum(0)).all()
    return y.detach()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dtype", [HF, BF])
def test_sums_beyond_the_largest_value(dtype, M, K, N, act):
    """Finite sums that the operands' type cannot hold: the slope is 0 or 1 there, as it is long before."""
    far = torch.tensor([-7e4, -1e5, 7e4, -3e6, 1e5, -65519.0, 65521.0] if dtype == HF else [-3.4e38, 3.4e38, -3.397e38, -1e30, 1e30], device=DEV)
    bias = far.repeat(N // far.numel() + 1)[:N]
    y = step(dtype, M, K, N, act, bias, bias > 0, 0.02)
    assert (y[:, bias < -7e4] == 0).all()


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dtype", [HF, BF])
def test_relu_of_sums_below_the_smallest_value(dtype, M, K, N):
    """A positive sum that rounds to zero in the operands' type has relu's slope of positive sums, a negative one or zero has none."""
    tiny = torch.tensor([2.0**-25, 1e-8, 2.0**-40, -1e-8, 0.0, -0.0, 1e-30, -(2.0**-25), 1.0, 3e-8] if dtype == HF else
                        [2.0**-134, 1e-41, -1e-41, 0.0, -0.0, 2.0**-149, -(2.0**-149), 1.0, 1e-38], device=DEV)
    bias = tiny.repeat(N // tiny.numel() + 1)[:N]
    step(dtype, M, K, N, "relu", bias, bias > 0, 0.0)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_sums_that_are_no_numbers_stay_so(dtype, act):
    x, w = torch.ones(4, 8, device=DEV, dtype=dtype), torch.zeros(16, 8, device=DEV, dtype=dtype)
    bias = torch.full((16,), float("nan"), device=DEV)
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    y = fg.fused_linear(*leaves, act)
    dx, dw, db = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert y.isnan().all() and dx.isnan().all() and dw.isnan().all() and db.isnan().all()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dtype", [HF, BF])
def test_infinite_sums_have_the_slope_of_the_limit(dtype, M, K, N, act):
    bias = torch.tensor([float("inf"), -float("inf"), 1e4, -1e4], device=DEV).repeat(N // 4 + 1)[:N]
    step(dtype, M, K, N, act, bias, bias > 0, 0.02)
