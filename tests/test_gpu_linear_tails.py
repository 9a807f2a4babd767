"""fused_linear: the activations far out on the negative side, held to a bound relative to the value.

The products are zeros, so that z is the fp32 bias.  exp(-s) is off by (2 + 1.173 s) 2^-23 of itself (the bound that CUDA documents for
its fast exponential) and by the roundings of s in fp32, s 2^-23; the rest of each formula by 2^-18.  Then one rounding: u of the
value, or half of the smallest subnormal, and 2^-140 for exponentials that are subnormal themselves."""

import pytest
import torch

import flaggems_vllm_b200 as fg

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_SUBNORMAL = {HF: 2.0**-25, BF: 2.0**-134, F32: 2.0**-150}
SIZES = [(1, 1024), (40, 1000), (2304, 1024)]


def relative(s):
    return (2 + 2.173 * s) * 2.0**-23 + 2.0**-18


def values(act, z, dtype, M, up=None):
    N = z.numel()
    x = torch.zeros(M, 16, device=DEV, dtype=dtype)
    bias = z if up is None else torch.cat([z, torch.full_like(z, up)])
    y = fg.fused_linear(x, torch.zeros(bias.numel(), 16, device=DEV, dtype=dtype), bias, act)
    assert y.shape == (M, N) and (y == y[:1]).all()
    return y[0].double()


def close(y, want, rel, dtype):
    bound = (torch.finfo(dtype).eps / 2 * (1 + rel) + rel) * want.abs() + HALF_SUBNORMAL[dtype] + 2.0**-140
    off = (y - want).abs()
    worst = (off / bound).argmax()
    assert (off <= bound).all(), f"{int((off > bound).sum())} beyond, worst {float((off / bound)[worst]):.3g} times, value {float(want[worst]):.3g}"


def gelu64(z):
    z = z.double()
    return z * 0.5 * torch.special.erfc(-z * 0.5**0.5)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N", SIZES)
def test_gelu(dtype, M, N):
    z = torch.linspace(-13.5, 8.0, N, device=DEV)
    close(values("gelu", z, dtype, M), gelu64(z), relative(z.double() ** 2 / 2), dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_slope_of_gelu(dtype):
    """Phi(z) + z phi(z) for z that the type holds, as the bias' gradient of one row; the two parts have opposite signs, so the bound is of
    the sum of their absolute values."""
    z = torch.linspace(-13.0, -0.5, 1000, device=DEV).to(dtype).float()
    x, bias = torch.zeros(1, 16, device=DEV, dtype=dtype), z.clone().requires_grad_()
    y = fg.fused_linear(x, torch.zeros(1000, 16, device=DEV, dtype=dtype), bias, "gelu")
    (db,) = torch.autograd.grad(y, bias, torch.ones_like(y))
    t = z.double()
    cdf, slope = 0.5 * torch.special.erfc(-t * 0.5**0.5), t * torch.exp(-t * t / 2) / (2 * torch.pi) ** 0.5
    off = (db.double() - (cdf + slope)).abs()
    assert (off <= relative(t * t / 2) * (cdf + slope.abs()) + 2.0**-140).all()


@pytest.mark.parametrize("act", ["silu", "silu_and_mul", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,N", SIZES)
def test_sigmoids(dtype, M, N, act):
    """z sigmoid(s): s = z, or for gelu_tanh s = 2 sqrt(2/pi) (z + 0.044715 z^3).  Down to exponentials of e^-100."""
    z = torch.linspace(-9.9 if act == "gelu_tanh" else -100.0, 20.0, N, device=DEV)
    t = z.double()
    s = t if act != "gelu_tanh" else 2 * (2 / torch.pi) ** 0.5 * (t + 0.044715 * t**3)
    want = t * torch.exp(s.clamp(max=0)) / (1 + torch.exp(-s.abs()))
    up = 0.75 if act == "silu_and_mul" else None
    roundings = 4.0 if act == "gelu_tanh" else 1.0  # its s is a polynomial in fp32
    close(values(act, z, dtype, M, up), want * (up or 1.0), relative(roundings * s.abs().clamp(max=110)), dtype)
