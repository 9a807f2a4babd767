"""The bytes of rms_norm_quant are those of a true division by the scale it returns, whatever the scale.

With rows of ones, eps = 0 and a length that is a power of two the norm is the weight, bit for bit (the mean square is exactly
one, and so is its root), so any fp32 values can be brought before the quantiser.  Zero tolerance: the values are placed on the
borders between neighbouring bytes and a few units of the last place to either side."""

import pytest
import torch

import flaggems_vllm_b200 as fg

pytestmark = pytest.mark.gpu

DEV = "cuda"
COLS, GROUP = 16384, 128
QMAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0, torch.int8: 127.0}


def borders(dtype):
    """The values half way between neighbours of the format, from its smallest on."""
    if dtype == torch.int8:
        return torch.arange(0, 127, device=DEV, dtype=torch.float32) + 0.5
    every = torch.arange(0, 256, dtype=torch.uint8, device=DEV).view(dtype).double()
    every = every[every.isfinite() & (every >= 0)].unique()
    return ((every[1:] + every[:-1]) / 2).float()


def shift(x, units):
    return (x.view(torch.int32) + units).view(torch.float32)


def bytes_of(exact, dtype):
    if dtype == torch.int8:
        return exact.round().clamp(-128, 127).to(torch.int8)
    return exact.clamp(max=QMAX[dtype]).to(dtype)


def check(w, dtype):
    """w: [groups, GROUP], what the quantiser gets."""
    x = torch.ones(1, COLS, device=DEV)
    assert torch.equal(fg.rms_norm(x, w.flatten(), 0.0)[0], w.flatten())
    q, s = fg.rms_norm_quant(x, w.flatten(), 0.0, group_size=GROUP, dtype=dtype, quant_eps=0.0)
    want = bytes_of(w / s.view(-1, 1), dtype)
    assert torch.equal(q.view(torch.uint8).view(w.shape), want.view(torch.uint8))
    return s.flatten()


@pytest.mark.parametrize("dtype", list(QMAX))
@pytest.mark.parametrize("exponent", [-120, -99, -96, -92, -88, -80, -70, -66, -40, 0, 60, 99, 110])
def test_scales_a_little_above_a_power_of_two(dtype, exponent):
    """There a remainder that lost its last bits turns a border into a tie."""
    n = COLS // GROUP
    s = shift(torch.full((n,), 2.0 ** exponent, device=DEV), torch.arange(n, device=DEV, dtype=torch.int32))
    inverse = torch.tensor(1.0 / QMAX[dtype], device=DEV)
    amax = shift((s * QMAX[dtype])[:, None], torch.arange(-2, 3, device=DEV, dtype=torch.int32))
    amax = amax.gather(1, (amax * inverse == s[:, None]).int().argmax(1, keepdim=True))  # the one that gives the scale, if any does
    units = torch.arange(-4, 5, device=DEV, dtype=torch.int32)
    edge = borders(dtype)[:14]
    w = torch.cat([amax, shift((s[:, None] * edge)[:, :, None], units).flatten(1), amax], 1)
    got = check(w, dtype)
    assert (got == s).float().mean() > 0.5


@pytest.mark.parametrize("dtype", list(QMAX))
@pytest.mark.parametrize("lo,hi", [(1e-37, 1e-33), (1e-30, 1e-26), (1e-21, 1e-19), (1e-3, 1e3), (1e28, 1e32)])
def test_scales_of_any_size(dtype, lo, hi):
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    edge, n = borders(dtype), COLS // GROUP
    for _ in range(20):
        s = (lo * (hi / lo) ** torch.rand((n, 1), generator=g, device=DEV, dtype=torch.float64)).float()
        at = torch.randint(0, edge.numel(), (n, GROUP), generator=g, device=DEV)
        w = shift(s * edge[at], torch.randint(-4, 5, (n, GROUP), generator=g, device=DEV, dtype=torch.int32))
        w[:, :1] = s * QMAX[dtype]  # the largest of the group
        check(w, dtype)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("cols", [256, 250])
def test_power_of_two_scales_have_a_floor(dtype, cols):
    """2^-33, the first power of two that is not below 1e-10, as the stand-alone quantiser has it, whatever quant_eps."""
    x = torch.ones(3, cols, device=DEV)
    for value in (0.0, 1e-30, 1e-10 * QMAX[dtype], 1.2e-10 * QMAX[dtype]):
        w = torch.full((cols,), value, device=DEV)
        want = 2.0 ** -32 if value == 1.2e-10 * QMAX[dtype] else 2.0 ** -33
        for quant_eps in (0.0, 1e-10 * value):
            q, s = fg.rms_norm_quant(x, w, 0.0, quant_eps=quant_eps, dtype=dtype, scale_ue8m0=True, group_size=cols // 2)
            assert (s == want).all()
            assert torch.equal(q.view(torch.uint8), bytes_of((w / want).expand_as(x), dtype).view(torch.uint8))
