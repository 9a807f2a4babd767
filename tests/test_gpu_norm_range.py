"""Norms and their gradients where fp32 itself is the limit: rows of tiny numbers and rows of millions of equal ones."""

import pytest
import torch

import flaggems_vllm_b200 as fg

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32 = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [64, 100, 1000, 1001, 1999, 2048, 2049, 4097, 7168, 20001, 33024])
def test_gradient_of_tiny_rows_without_eps(cols, dtype):
    """Rows of some 2^-65: the squares are normal numbers (2^-130 is a subnormal of 19 bits), the square of the root's inverse is
    infinite.  Alignment and length do not matter."""
    g = torch.Generator(device=DEV)
    g.manual_seed(cols)
    sign = torch.randint(0, 2, (5, cols), generator=g, device=DEV) * 2 - 1
    x = ((1.0 + torch.rand((5, cols), generator=g, device=DEV)) * sign * 2.0 ** -65).to(dtype)
    w = (1.0 + 0.5 * torch.rand((cols,), generator=g, device=DEV)).to(dtype)
    dy = torch.randn((5, cols), generator=g, device=DEV).to(dtype)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fg.rms_norm(xl, wl, 0.0)
    dx, dw = torch.autograd.grad(y, (xl, wl), dy)
    xd, wd, dyd = x.double(), w.double(), dy.double()
    inv = 1.0 / xd.square().mean(-1, keepdim=True).sqrt()
    n = xd * inv
    mean = (wd * dyd * n).mean(-1, keepdim=True)
    want = inv * (wd * dyd - n * mean)
    # squares are off by 2^-19 at most, their root by half of that, and so is what is made of it; each sum adds its additions'
    off = 2.0 ** -20 + (cols // 256 + 80) * F32
    half = torch.finfo(dtype).eps / 2
    assert ((y.double() - n * wd).abs() <= (n * wd).abs() * (half + off)).all()
    size = inv * ((wd * dyd).abs() + n.abs() * (wd * dyd * n).abs().mean(-1, keepdim=True) * 2)
    assert ((dx.double() - want).abs() <= want.abs() * half + size * 2 * off).all()
    dww = (dyd * n).sum(0)
    assert ((dw.double() - dww).abs() <= dww.abs() * half + (dyd * n).abs().sum(0) * (off + 16 * F32) + 1e-38).all()


@pytest.mark.parametrize("cols", [33024, (1 << 20) + 8, (1 << 22) + 1, 1 << 24])
@pytest.mark.parametrize("residual", [False, True])
def test_long_rows_of_equal_numbers(cols, residual):
    """The errors of additions do not cancel here; those of a row's sums must not grow with its length: at most 32 terms and a
    tree of 8 additions are fp32, and each product, quotient, root and rounding counts one."""
    value = 1.1
    x = torch.full((1, cols), value, device=DEV)
    r = torch.full((1, cols), 0.0, device=DEV) if residual else None
    w = torch.full((cols,), 1.3, device=DEV)
    leaves = [t.requires_grad_() for t in (x, w)]
    out = fg.rms_norm(*leaves, 0.0, r)
    y = out[0] if residual else out
    sums = 32 + 8 + 2
    want = float(w.detach()[0].double())  # x / |x| times the weight
    assert abs(y.double() - want).max().item() <= want * (sums / 2 + 5) * F32
    # dy = 1 in one half, 3 in the other: dx = r w (dy - 2), where the mean of dy is 2 but for the odd column
    dy = torch.ones_like(y)
    dy[:, cols // 2:] = 3.0
    dx, _ = torch.autograd.grad(y, leaves, dy)
    mean = 1.0 + 2.0 * (cols - cols // 2) / cols
    inv = 1.0 / float(x.detach()[0, 0].double())
    exact = (inv * want * (dy.double() - mean))
    # terms of the size r w dy and r w mean, each off by its own share: half the first sum's for r, three halves and the second sum's
    off = inv * want * (3.0 * (sums / 2 + 5) + mean * (2.5 * sums + 12)) * F32
    assert (dx.double() - exact).abs().max().item() <= off


@pytest.mark.parametrize("rows,cols", [(40, 1 << 22), (40, (1 << 22) + 1), (70, (1 << 20) + 3)])
def test_gradient_of_more_rows_than_parts(rows, cols):
    """Long rows share 16 parts of the weight's gradient, or as many as 256 MB hold."""
    g = torch.Generator(device=DEV)
    g.manual_seed(rows)
    x = torch.randn((rows, cols), generator=g, device=DEV).bfloat16()
    dy = torch.randn((rows, cols), generator=g, device=DEV).bfloat16()
    xl, wl = x.clone().requires_grad_(), torch.ones(cols, device=DEV, requires_grad=True)
    dx, dw = torch.autograd.grad(fg.rms_norm(xl, wl), (xl, wl), dy)
    want, terms = torch.zeros(cols, dtype=torch.float64, device=DEV), torch.zeros(cols, dtype=torch.float64, device=DEV)
    off = (32 + 8 + 2) / 2 + 6 + rows  # a row's sum and root, its products; then every row behind one another at most
    for i in range(rows):
        n = x[i].double() / (x[i].double().square().mean() + 1e-6).sqrt()
        want += n * dy[i].double()
        terms += (n * dy[i].double()).abs()
        exact = (dy[i].double() - n * (n * dy[i].double()).mean()) / (x[i].double().square().mean() + 1e-6).sqrt()
        # a mean of products of random signs; its error is counted on their magnitudes
        tol = exact.abs() * 2.0 ** -8 + (dy[i].double().abs() + n.abs()) * 2 * (off + 64) * F32
        assert ((dx[i].double() - exact).abs() <= tol).all()
    assert ((dw.double() - want).abs() <= terms * off * F32 + 1e-38).all()
